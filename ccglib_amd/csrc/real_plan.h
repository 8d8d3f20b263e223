// Which block shape a real product runs as, and into how many parts its K is cut.
#ifndef CCGLIB_AMD_REAL_PLAN_H_
#define CCGLIB_AMD_REAL_PLAN_H_

#include <algorithm>

#include "scaled.h"

namespace ccglib_amd {

inline size_t real_blocks(const RealShape &s, size_t batch, size_t nx, size_t ny, bool symmetric) {
  const size_t y = ceil_div(ny, s.by);
  return batch * (symmetric ? y * (y + 1) / 2 : ceil_div(nx, s.bx) * y);
}

inline RealGemmPlan plan_real_gemm(const RealShape *shapes, int count, size_t batch, size_t nx, size_t ny, size_t pieces,
                                   bool symmetric) {
  constexpr size_t kUnits = 256;
  RealGemmPlan plan;
  pieces = std::max<size_t>(1, pieces);
  size_t parts = 0;
  if (real_block_option) {
    plan.shape = (int)std::min<size_t>(real_block_option % 256 - 1, count - 1);
    parts = real_block_option / 256;
  } else if (count == 4 && ny <= 32) {
    plan.shape = 3;
  } else {
    for (int s = 0; s < 3 && s < count; ++s) {
      plan.shape = s;
      if (real_blocks(shapes[s], batch, nx, ny, symmetric) >= (s == 0 ? kUnits : kUnits / 2)) break;
    }
  }
  const RealShape &s = shapes[plan.shape];
  const size_t blocks = real_blocks(s, batch, nx, ny, symmetric);
  if (parts == 0) {
    parts = 1;
    while (blocks * parts < kUnits && pieces / (parts * 2) >= 4) parts *= 2;
  }
  parts = std::min(parts, pieces);
  plan.pieces_per_part = (unsigned)ceil_div(pieces, parts);
  plan.parts = (unsigned)ceil_div(pieces, (size_t)plan.pieces_per_part);
  if (plan.parts > 1) {
    plan.partial_bytes = blocks * plan.parts * s.bx * s.by * sizeof(float);
    plan.counter_bytes = blocks * sizeof(unsigned);
  }
  return plan;
}

}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_REAL_PLAN_H_
