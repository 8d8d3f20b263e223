// C entry point to what a ScaledLinear hands its kernels, without a GPU: the launchers are recorded instead of run.
#include "../../ccglib_amd/csrc/scaled_gemm.hip"
#include "../../ccglib_amd/csrc/scaled_linear.h"

namespace ccglib_amd {
size_t real_block_option = 0;
namespace real {
static Args g_args;
#define CCGLIB_RECORDED(MODE)                                                                          \
  template <> hipError_t launch_scaled_mode<MODE>(const ScaledGemmParams &, const Args &a, hipStream_t) { \
    g_args = a;                                                                                        \
    return hipSuccess;                                                                                 \
  }
CCGLIB_RECORDED(kScaledBlocks)
CCGLIB_RECORDED(kScaledRows)
CCGLIB_RECORDED(kScaledE8m0)
CCGLIB_RECORDED(kWideBlocks)
CCGLIB_RECORDED(kWideRows)
CCGLIB_RECORDED(kWideE8m0)
#undef CCGLIB_RECORDED
}  // namespace real
}  // namespace ccglib_amd

using namespace ccglib_amd;

// ranges: counters and partial sums (begin, end) of the three products, empty where K is in one part, then values and scales
// of the six copies; sizes: of the memory, and of what is cleared in it. Offsets into the memory.
extern "C" void scaled_linear_layout(size_t M, size_t N, size_t K, int type, int gradient_type, int scale_type, size_t option,
                                     size_t *ranges, size_t *sizes) {
  real_block_option = option;
  ScaledLinearParams l = scaled_linear_params(M, N, K, type, gradient_type, scale_type, true);
  plan_scaled_linear(&l);
  char *const base = reinterpret_cast<char *>((uintptr_t)1 << 40);
  place_scaled_linear(&l, base);
  auto put = [&](const void *from, size_t bytes) {
    *ranges++ = (size_t)(static_cast<const char *>(from) - base);
    *ranges++ = (size_t)(static_cast<const char *>(from) - base) + bytes;
  };
  for (const ScaledGemmParams *p : {&l.y, &l.dx, &l.dw}) {
    real::g_args = {};
    (void)launch_scaled_gemm(*p, nullptr);
    const real::Args &a = real::g_args;
    const RealShape &shape = shapes_of(*p)[p->plan.shape];
    const size_t blocks = a.parts > 1 ? (size_t)a.batch * a.blocks_x * a.blocks_y : 0;
    put(a.arrived, blocks * sizeof *a.arrived);
    put(a.partial, blocks * a.parts * shape.bx * shape.by * sizeof *a.partial);
  }
  for (const QuantizeParams *p : {&l.x, &l.w, &l.dy}) {
    put(p->out, p->m * scaled_pitch(p->n));
    put(p->scales, ceil_div(p->n, kScaleGroup) * scaled_pitch(scale_rows(p->m, p->group)) * scale_size(p->scale_type));
    put(p->out_t, p->n * scaled_pitch(p->m));
    put(p->scales_t, ceil_div(p->m, kScaleGroup) * scaled_pitch(scale_rows(p->n, p->group)) * scale_size(p->scale_type));
  }
  sizes[0] = l.bytes;
  sizes[1] = l.counter_bytes;
}
