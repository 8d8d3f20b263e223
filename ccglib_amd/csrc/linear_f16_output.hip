// 16-bit linear layers: the kernels of one type and product (see linear_gemm.h)
#define CCGLIB_LINEAR_TYPE kFloat16
#define CCGLIB_LINEAR_KIND kOutput
#include "linear_gemm.h"
