// 8-bit products with block scales: which kernel a product runs as, and its launch (kernels: scaled_gemm.h).
#include <algorithm>
#include <cstdio>

#include "real_plan.h"
#include "scaled_gemm.h"

namespace ccglib_amd {
namespace {

constexpr RealShape kShapes[2][4] = {
#define CCGLIB_INFO(ID, BX, BY, WX, WY, SLOTS, EU) {BX, BY, 64 * WX * WY, #BY "x" #BX},
    {CCGLIB_SCALED_SHAPES(CCGLIB_INFO)},
    {CCGLIB_WIDE_SHAPES(CCGLIB_INFO)}
#undef CCGLIB_INFO
};

bool is_wide(const ScaledGemmParams &p) { return p.type_c == kFloat32; }

int mode_of(const ScaledGemmParams &p) {
  const int mode = p.scale_type == kScaleE8m0 ? real::kScaledE8m0 : p.group_b == kScaleBlocks ? real::kScaledBlocks : real::kScaledRows;
  return is_wide(p) ? mode + real::kWideBlocks : mode;
}

}  // namespace

RealGemmPlan plan_scaled_gemm(const ScaledGemmParams &p) {
  return plan_real_gemm(kShapes[is_wide(p)], 4, p.batch, p.n, p.m, ceil_div(p.k, (size_t)real::kPieceBytes), false);
}

const char *describe_scaled_gemm(const ScaledGemmParams &p) {
  static thread_local char name[96];
  static const char *const scales[] = {"float scales, 128 x 128", "float scales", "e8m0 scales"};
  snprintf(name, sizeof name, "gemm_real<8 bits%s, %s> %s block, K in %u", is_wide(p) ? " as fp16" : "", scales[mode_of(p) % 3],
           kShapes[is_wide(p)][p.plan.shape].name, p.plan.parts);
  return name;
}

hipError_t launch_scaled_gemm(const ScaledGemmParams &p, hipStream_t stream) {
  if (p.batch == 0 || p.m == 0 || p.n == 0) return hipSuccess;
  const RealShape &shape = kShapes[is_wide(p)][p.plan.shape];
  const int mode = mode_of(p);
  real::Args a = {};
  a.x = static_cast<const char *>(p.b);
  a.y = static_cast<const char *>(p.a);
  a.nx = p.n;
  a.ny = p.m;
  a.batch = p.batch;
  a.x_pitch = (unsigned)p.pitch_b;
  a.y_pitch = (unsigned)p.pitch_a;
  a.x_batch = (size_t)p.n * p.pitch_b;
  a.y_batch = (size_t)p.m * p.pitch_a;
  a.k_bytes = (unsigned)scaled_pitch(p.k);
  a.pieces = (unsigned)ceil_div(p.k, (size_t)real::kPieceBytes);
  a.blocks_x = (unsigned)ceil_div(p.n, shape.bx);
  a.blocks_y = (unsigned)ceil_div(p.m, shape.by);
  a.x_scales = static_cast<const char *>(p.scales_b);
  a.y_scales = static_cast<const char *>(p.scales_a);
  a.x_scale_pitch = (unsigned)scaled_pitch(scale_rows(p.n, p.group_b));
  a.y_scale_pitch = (unsigned)scaled_pitch(scale_rows(p.m, p.group_a));
  a.x_shift = p.group_b == kScaleBlocks ? 7 : 0;
  a.y_shift = p.group_a == kScaleBlocks ? 7 : 0;
  a.parts = p.plan.parts;
  a.pieces_per_part = p.plan.pieces_per_part;
  a.arrived = static_cast<unsigned *>(p.workspace);
  a.partial = reinterpret_cast<float *>(static_cast<char *>(p.workspace) + ceil_div(p.plan.counter_bytes, 256) * 256);
  switch (mode) {
    case real::kScaledBlocks: return real::launch_scaled_mode<real::kScaledBlocks>(p, a, stream);
    case real::kScaledRows: return real::launch_scaled_mode<real::kScaledRows>(p, a, stream);
    case real::kScaledE8m0: return real::launch_scaled_mode<real::kScaledE8m0>(p, a, stream);
    case real::kWideBlocks: return real::launch_scaled_mode<real::kWideBlocks>(p, a, stream);
    case real::kWideRows: return real::launch_scaled_mode<real::kWideRows>(p, a, stream);
    default: return real::launch_scaled_mode<real::kWideE8m0>(p, a, stream);
  }
}

}  // namespace ccglib_amd
