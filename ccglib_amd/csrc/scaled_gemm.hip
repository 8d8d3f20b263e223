// 8-bit products with block scales: which kernel a product runs as, and its launch (kernels: scaled_gemm.h).
#include <algorithm>
#include <cstdio>

#include "real_plan.h"
#include "scaled_gemm.h"

namespace ccglib_amd {
namespace {

// (the shapes of scaled_gemm.h, in their order; see real_plan.h for the figures)
constexpr RealShape kBlocksShapes[] = {{256, 256, 512, 1, 0.92f, 1.79f, 8.0f, 0.69f, "256x256"},
                                       {128, 128, 256, 2, 0.81f, 1.07f, 4.2f, 1.06f, "128x128"},
                                       {64, 64, 256, 2, 0.243f, 0.442f, 2.5f, 2.4f, "64x64"},
                                       {64, 32, 256, 2, 0.181f, 0.33f, 2.7f, 4.5f, "32x64"},
                                       {128, 128, 512, 1, 0.45f, 0.62f, 3.4f, 0.92f, "128x128 8-wave"},
                                       {192, 192, 512, 1, 0.78f, 1.27f, 5.6f, 0.96f, "192x192"}};
constexpr RealShape kRowsShapes[] = {{256, 256, 512, 1, 1.16f, 2.17f, 8.6f, 0.82f, "256x256"},
                                     {128, 128, 256, 2, 0.88f, 1.25f, 4.3f, 1.15f, "128x128"},
                                     {64, 64, 256, 2, 0.278f, 0.481f, 2.6f, 2.4f, "64x64"},
                                     {64, 32, 256, 2, 0.206f, 0.356f, 2.5f, 4.6f, "32x64"},
                                     {128, 128, 512, 1, 0.55f, 0.69f, 3.9f, 0.88f, "128x128 8-wave"},
                                     {192, 192, 512, 1, 0.82f, 1.25f, 5.7f, 0.95f, "192x192"}};
constexpr RealShape kE8m0Shapes[] = {{256, 256, 512, 1, 0.84f, 1.56f, 7.8f, 0.74f, "256x256"},
                                     {128, 128, 256, 2, 0.76f, 0.95f, 4.8f, 1.23f, "128x128"},
                                     {64, 64, 256, 2, 0.213f, 0.433f, 2.3f, 2.5f, "64x64"},
                                     {64, 32, 256, 2, 0.164f, 0.306f, 3.2f, 5.4f, "32x64"},
                                     {128, 128, 512, 1, 0.38f, 0.53f, 3.6f, 1.05f, "128x128 8-wave"},
                                     {192, 192, 512, 1, 0.57f, 0.89f, 5.9f, 0.92f, "192x192"}};
constexpr RealShape kWideShapes[] = {{128, 256, 512, 1, 1.34f, 1.97f, 8.5f, 0.98f, "256x128"},
                                     {128, 128, 256, 2, 1.13f, 1.97f, 7.1f, 1.73f, "128x128"},
                                     {64, 64, 256, 2, 0.459f, 0.758f, 2.9f, 2.4f, "64x64"},
                                     {64, 32, 256, 2, 0.304f, 0.505f, 2.6f, 4.1f, "32x64"},
                                     {128, 128, 512, 1, 0.87f, 1.24f, 5.4f, 1.08f, "128x128 8-wave"}};
constexpr int kShapes = sizeof kBlocksShapes / sizeof kBlocksShapes[0], kWideCount = sizeof kWideShapes / sizeof kWideShapes[0];
#define CCGLIB_SAME(ID, BX, BY, WX, WY, SLOTS, EU) \
  static_assert(CCGLIB_TABLE[ID].bx == BX && CCGLIB_TABLE[ID].by == BY && CCGLIB_TABLE[ID].threads == 64 * WX * WY, \
                "the table is in the order of the shapes");
#define CCGLIB_TABLE kBlocksShapes
CCGLIB_SCALED_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#define CCGLIB_TABLE kRowsShapes
CCGLIB_SCALED_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#define CCGLIB_TABLE kE8m0Shapes
CCGLIB_SCALED_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#define CCGLIB_TABLE kWideShapes
CCGLIB_WIDE_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#undef CCGLIB_SAME

bool is_wide(const ScaledGemmParams &p) { return p.type_c == kFloat32; }

int mode_of(const ScaledGemmParams &p) {
  const int mode = p.scale_type == kScaleE8m0 ? real::kScaledE8m0 : p.group_b == kScaleBlocks ? real::kScaledBlocks : real::kScaledRows;
  return is_wide(p) ? mode + real::kWideBlocks : mode;
}

const RealShape *shapes_of(const ScaledGemmParams &p) {
  if (is_wide(p)) return kWideShapes;
  return p.scale_type == kScaleE8m0 ? kE8m0Shapes : p.group_b == kScaleBlocks ? kBlocksShapes : kRowsShapes;
}

}  // namespace

RealGemmPlan plan_scaled_gemm(const ScaledGemmParams &p) {
  return plan_real_gemm(shapes_of(p), is_wide(p) ? kWideCount : kShapes, p.batch, p.n, p.m, ceil_div(p.k, (size_t)real::kPieceBytes), false, real_block_option);
}

bool scaled_gemm_launches(const ScaledGemmParams &p) {
  const RealShape &shape = shapes_of(p)[p.plan.shape];
  return real_launches(shape, real_blocks(shape, p.batch, p.n, p.m, false) * p.plan.parts);
}

const char *describe_scaled_gemm(const ScaledGemmParams &p) {
  static thread_local char name[96];
  static const char *const scales[] = {"float scales, 128 x 128", "float scales", "e8m0 scales"};
  snprintf(name, sizeof name, "gemm_real<8 bits%s, %s> %s block, K in %u", is_wide(p) ? " as fp16" : "", scales[mode_of(p) % 3],
           shapes_of(p)[p.plan.shape].name, p.plan.parts);
  return name;
}

hipError_t launch_scaled_gemm(const ScaledGemmParams &p, hipStream_t stream) {
  if (p.batch == 0 || p.m == 0 || p.n == 0) return hipSuccess;
  const RealShape &shape = shapes_of(p)[p.plan.shape];
  int mode = mode_of(p);
  // (a wave of such a block has columns of two scales)
  if (mode == real::kScaledBlocks && shape.bx % 128 != 0 && 128 % shape.bx != 0) mode = real::kScaledRows;
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
  a.arrived = p.arrived;
  a.partial = p.partial;
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
