// Umbrella header of the ccglib-compatible C++ API for gfx950.
#ifndef CCGLIB_CCGLIB_HPP_
#define CCGLIB_CCGLIB_HPP_
#include <ccglib/gemm/mma.h>
#include <ccglib/gemm/reference.h>
#include <ccglib/gemm/scaled_gemm.h>
#include <ccglib/orthogonalize/orthogonalize.h>
#include <ccglib/packing/packing.h>
#include <ccglib/pipeline/fused_linear.h>
#include <ccglib/pipeline/grouped_linear.h>
#include <ccglib/pipeline/pipeline.h>
#include <ccglib/pipeline/scaled_linear.h>
#include <ccglib/quantize/quantize.h>
#include <ccglib/route/route.h>
#include <ccglib/transpose/transpose.h>
#endif
