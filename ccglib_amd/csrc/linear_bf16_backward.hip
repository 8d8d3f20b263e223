// 16-bit linear layers: the kernels of small backward passes of one type (see linear_backward.h)
#define CCGLIB_LINEAR_TYPE kBfloat16
#include "linear_backward.h"
