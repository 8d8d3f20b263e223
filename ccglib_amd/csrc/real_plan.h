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

// Whether a launch takes so many blocks: with 2^32 work-items or more it is no error to the runtime, but starts what is left
// of their number modulo 2^32.
inline bool real_launches(const RealShape &s, size_t blocks) { return blocks <= 0xffffffffu / s.threads; }

// The time of a product as that of its busiest unit: rounds of blocks, all units full in all but the last one. The figures of the
// 8-bit products were fitted to 38 problems from 1 x 8192 x 8192 to 8192 x 4096 x 4096 in every shape and 1 to 32 parts. On 30 other
// problems, most of them small, the choice is behind the fastest shape and number of parts by 2.1 and 1.5 % (float scales of blocks and
// rows), 3.2 % (e8m0) and 1.5 % (32-bit C) in the mean, and by 5 to 11 % where it is wrong (3000 x 3000 x 8192 with 32-bit C: 22 %). The
// figures of the updates are estimates from a trace: whole updates of 12 sizes are 0.3 % (bf16) and 1.5 % (float32) in the mean, 8 % at
// most, behind the fastest single shape for all of their products.
inline double real_gemm_us(const RealShape &s, size_t blocks, size_t pieces, size_t parts) {
  constexpr size_t kUnits = 256;
  const double per_part = (double)ceil_div(pieces, parts);
  const size_t all = blocks * parts, slots = kUnits * s.per_unit, rounds = all / slots, rest = all % slots;
  double us = (double)rounds * (per_part * s.full_us + s.block_us);
  if (rest) {
    double piece = s.full_us;                       // (some unit has two blocks)
    if (rest <= kUnits) {
      piece = s.alone_us;
      // (one block a unit: the more units, the lower the clock)
      if (s.per_unit == 1) piece += (s.full_us - s.alone_us) * (double)rest / (double)kUnits;
    }
    us += per_part * piece + s.block_us;
  }
  if (parts > 1) us += s.join_us * (1.0 + 0.25 * (double)parts) * s.bx * s.by / 4096.0;
  return us;
}

// option: REAL_BLOCK
inline RealGemmPlan plan_real_gemm(const RealShape *shapes, int count, size_t batch, size_t nx, size_t ny, size_t pieces,
                                   bool symmetric, size_t option) {
  RealGemmPlan plan;
  pieces = std::max<size_t>(1, pieces);
  const int first = option ? (int)std::min<size_t>(option % 256 - 1, count - 1) : 0;
  const int end = option ? first + 1 : count;
  double best = 0.0;
  size_t parts = 0;
  for (int s = first; s < end; ++s) {
    const size_t blocks = real_blocks(shapes[s], batch, nx, ny, symmetric);
    for (size_t p : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (p > pieces) break;
      if (!real_launches(shapes[s], blocks * p)) break;
      const double us = real_gemm_us(shapes[s], blocks, pieces, p);
      if (parts == 0 || us < best) {
        best = us;
        parts = p;
        plan.shape = s;
      }
      if (blocks * p > 65536) break;                // (more parts of so many blocks: nothing but memory)
    }
  }
  if (parts == 0) parts = 1;                        // (no shape has few enough blocks: scaled_gemm_launches says so)
  if (option / 256) parts = std::min(option / 256, pieces);
  const RealShape &s = shapes[plan.shape];
  const size_t blocks = real_blocks(s, batch, nx, ny, symmetric);
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
