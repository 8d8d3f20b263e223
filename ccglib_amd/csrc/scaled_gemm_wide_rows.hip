// 8-bit products with block scales: the kernels of one kind of scale, 32-bit C (see scaled_gemm.h)
#define CCGLIB_SCALED_MODE 4
#include "scaled_gemm.h"
