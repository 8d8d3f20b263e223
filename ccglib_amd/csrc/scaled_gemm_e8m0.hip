// 8-bit products with block scales: the kernels of one kind of scale (see scaled_gemm.h)
#define CCGLIB_SCALED_MODE 2
#include "scaled_gemm.h"
