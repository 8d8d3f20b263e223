// The three products and the conversions of a ScaledLinear, and where in its one allocation each has its memory.
#ifndef CCGLIB_AMD_SCALED_LINEAR_H_
#define CCGLIB_AMD_SCALED_LINEAR_H_

#include <algorithm>
#include <cstdint>

#include "scaled.h"

namespace ccglib_amd {

inline size_t scale_size(int scale_type) { return scale_type == kScaleE8m0 ? 1 : 4; }

struct ScaledLinearParams {
  QuantizeParams x, w, dy;
  ScaledGemmParams y, dx, dw;
  bool training;
  size_t counter_bytes, bytes;      // of the memory: what is cleared first (from its start), all of it
};

// Sizes and types, no plans and no memory yet.
inline ScaledLinearParams scaled_linear_params(size_t M, size_t N, size_t K, int type, int gradient_type, int scale_type, bool training) {
  auto quantize = [&](size_t m, size_t n, int out, int group) {
    QuantizeParams p = {};
    p.batch = 1;
    p.m = (unsigned)m;
    p.n = (unsigned)n;
    p.in_pitch = n;
    p.type_in = type;
    p.type_out = out;
    p.group = group;
    p.scale_type = scale_type;
    return p;
  };
  auto gemm = [&](size_t m, size_t n, size_t k, int a, int c, int group_b) {
    ScaledGemmParams p = {};
    p.batch = 1;
    p.m = (unsigned)m;
    p.n = (unsigned)n;
    p.k = (unsigned)k;
    p.pitch_a = p.pitch_b = scaled_pitch(k);
    p.pitch_c = n;
    p.type_a = a;
    p.type_b = kFloat8e4m3;
    p.type_c = c;
    p.group_a = kScaleRows;
    p.group_b = group_b;
    p.scale_type = scale_type;
    return p;
  };
  ScaledLinearParams l = {};
  l.training = training;
  l.x = quantize(M, K, kFloat8e4m3, kScaleRows);
  l.w = quantize(N, K, kFloat8e4m3, kScaleBlocks);
  l.dy = quantize(M, N, gradient_type, kScaleRows);
  l.y = gemm(M, N, K, kFloat8e4m3, type, kScaleBlocks);
  l.dx = gemm(M, K, N, gradient_type, type, kScaleBlocks);
  l.dw = gemm(N, K, M, gradient_type, kFloat32, kScaleRows);
  return l;
}

inline void plan_scaled_linear(ScaledLinearParams *l) {
  l->y.plan = plan_scaled_gemm(l->y);
  if (l->training) {
    l->dx.plan = plan_scaled_gemm(l->dx);
    l->dw.plan = plan_scaled_gemm(l->dw);
  }
}

// Points everything into `memory` (null: to learn `bytes` and `counter_bytes`). The products run one after the other and share
// counters and partial sums: all counters lie in front of all sums, however many of either a product has, since a product's
// counters have to be zero when it starts, whatever ran before it. Behind them the 8-bit copies of x, w and dy in both
// orientations (without training: of x and w as they are).
inline void place_scaled_linear(ScaledLinearParams *l, char *memory) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *const here = reinterpret_cast<char *>(reinterpret_cast<uintptr_t>(memory) + at);
    at += ceil_div(bytes, 256) * 256;
    return here;
  };
  ScaledGemmParams *const products[] = {&l->y, &l->dx, &l->dw};
  const int count = l->training ? 3 : 1;
  size_t counters = 0, sums = 0;
  for (int i = 0; i < count; ++i) {
    counters = std::max(counters, products[i]->plan.counter_bytes);
    sums = std::max(sums, products[i]->plan.partial_bytes);
  }
  unsigned *const arrived = reinterpret_cast<unsigned *>(take(counters));
  float *const partial = reinterpret_cast<float *>(take(sums));
  for (int i = 0; i < count; ++i) {
    products[i]->arrived = arrived;
    products[i]->partial = partial;
  }
  struct Copy {
    char *values, *scales;
  };
  auto copy = [&](const QuantizeParams &p, bool transposed) {
    const size_t rows = transposed ? p.n : p.m, k = transposed ? p.m : p.n;
    Copy c;
    c.values = take(rows * scaled_pitch(k));
    c.scales = take(ceil_div(k, kScaleGroup) * scaled_pitch(scale_rows(rows, p.group)) * scale_size(p.scale_type));
    return c;
  };
  auto keep = [&](QuantizeParams *p, ScaledGemmParams *gemm, bool as_a, ScaledGemmParams *gemm_t, bool as_a_t) {
    auto give = [](ScaledGemmParams *to, bool a, const Copy &c) {
      (a ? to->a : to->b) = c.values;
      (a ? to->scales_a : to->scales_b) = c.scales;
    };
    const Copy direct = copy(*p, false);
    p->out = direct.values;
    p->scales = direct.scales;
    give(gemm, as_a, direct);
    if (l->training) {
      const Copy transposed = copy(*p, true);
      p->out_t = transposed.values;
      p->scales_t = transposed.scales;
      give(gemm_t, as_a_t, transposed);
    }
  };
  keep(&l->x, &l->y, true, &l->dw, false);      // y = x W^T, dw = dy^T x
  keep(&l->w, &l->y, false, &l->dx, false);     // dx = dy W
  if (l->training) keep(&l->dy, &l->dx, true, &l->dw, true);
  l->counter_bytes = counters;
  l->bytes = at;
}

}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_SCALED_LINEAR_H_
