// The products of a small layer's backward pass in one launch: dx, dW and the last sums of dbias need nothing of each other, and
// each of them alone leaves units idle. A workgroup has a block of one of them. (300 x 255 x 577 with dbias: 18.8 us in launches of their
// own, 11.0 together; 512 x 512 x 512: dx 6.8, dW 6.1, both 6.8.)
#ifndef CCGLIB_AMD_LINEAR_BACKWARD_H_
#define CCGLIB_AMD_LINEAR_BACKWARD_H_

#include "linear_gemm.h"

namespace ccglib_amd {
namespace linear {

// What the column sums of dz are made in: blocks of columns, and of rows of a group. Few rows a block where many would leave units idle: a wave's
// loads are on their way together then (300 x 255: 12.8 us with 64 rows, 5.2 with 16).
constexpr unsigned kGradientColumns = 512, kFewRows = 16, kManyRows = 64;

// dbias (+)= the sums of a group's row blocks. Workgroup `block` has 64 columns of a group, each of its first four waves a quarter of the blocks, in
// their order (256 columns, all blocks a wave: 8.8 us for 128 blocks of 4096 columns, 4.7 like this).
constexpr unsigned kJoinColumns = 64;
struct JoinArgs {
  const float *sums;
  char *db;
  unsigned n, rows, blocks;      // blocks: of rows, as many as there can be
  unsigned few;                  // they have kFewRows rows, else kManyRows
  int type, accumulate;
  const int *offsets;
  unsigned groups;
};
template <unsigned ROWS> __device__ __forceinline__ void join_blocks(const JoinArgs &a, float *lds, unsigned x, unsigned group) {
  unsigned from = 0, count = (a.rows + ROWS - 1) / ROWS;
  if (a.offsets) {
    if (group > 0) from = RowBlocks<ROWS>(a.offsets, group, a.rows).all();
    count = (span_of(a.offsets, group, a.rows).count + ROWS - 1) / ROWS;
  }
  if (from > a.blocks) from = a.blocks;      // (offsets that fall: no sums are read that nobody can have written)
  if (count > a.blocks - from) count = a.blocks - from;
  const unsigned wave = threadIdx.x / 64, lane = threadIdx.x % 64, share = (count + 3) / 4;
  const unsigned first = wave * share, until = first + share < count ? first + share : count;
  float sum = 0.f;
  if (wave < 4 && x < a.n) {
#pragma unroll 8
    for (unsigned b = first; b < until; ++b) sum += a.sums[(size_t)(from + b) * a.n + x];
    lds[wave * 64 + lane] = sum;
  }
  __syncthreads();
  if (wave > 0 || x >= a.n) return;
  sum = (sum + lds[64 + lane]) + (lds[128 + lane] + lds[192 + lane]);
  const size_t at = (size_t)group * a.n + x;
  if (a.type == kFloat32) {
    float *const db = reinterpret_cast<float *>(a.db) + at;
    *db = a.accumulate ? *db + sum : sum;
  } else if (a.type == kFloat16) {
    reinterpret_cast<_Float16 *>(a.db)[at] = (_Float16)sum;
  } else {
    reinterpret_cast<__bf16 *>(a.db)[at] = (__bf16)sum;
  }
}
inline size_t join_workgroups(size_t n, size_t groups) { return ceil_div(n, (size_t)kJoinColumns) * groups; }
// lds: 1 KiB
__device__ __forceinline__ void join(const JoinArgs &a, float *lds, unsigned block) {
  const unsigned across = (a.n + kJoinColumns - 1) / kJoinColumns, group = block / across;
  const unsigned x = (block - group * across) * kJoinColumns + threadIdx.x % 64;
  if (a.few) {
    join_blocks<kFewRows>(a, lds, x, group);
  } else {
    join_blocks<kManyRows>(a, lds, x, group);
  }
}

struct BackwardArgs {
  Args input, weights;
  StoreParams store_input, store_weights;
  JoinArgs join;
  unsigned input_blocks, weights_blocks;   // workgroups: those of the input's gradient, of the weights', then those of join
};

template <int TYPE, int BX, int BY, int WX, int WY, int SLOTS, int WAVES_PER_EU>
__global__ __launch_bounds__(64 * WX * WY, WAVES_PER_EU) void gemm_linear_backward(BackwardArgs a) {
  __shared__ __attribute__((aligned(256))) char lds[kLdsBytes<BX, BY, SLOTS>];
  const unsigned id = blockIdx.x;
  if (id < a.input_blocks) {
    product<TYPE, kInput, BX, BY, WX, WY, SLOTS>(a.input, a.store_input, lds, id, a.input_blocks);
  } else if (id - a.input_blocks < a.weights_blocks) {
    product<TYPE, kWeights, BX, BY, WX, WY, SLOTS>(a.weights, a.store_weights, lds, id - a.input_blocks, a.weights_blocks);
  } else {
    join(a.join, reinterpret_cast<float *>(lds), id - a.input_blocks - a.weights_blocks);
  }
}

// The shapes of linear_gemm.h that it comes in
constexpr bool backward_in_one(int shape) { return shape >= 1 && shape <= 3; }

template <int TYPE> hipError_t launch_backward(int shape, unsigned grid, const BackwardArgs &a, hipStream_t stream);
template <> hipError_t launch_backward<kFloat16>(int shape, unsigned grid, const BackwardArgs &a, hipStream_t stream);
template <> hipError_t launch_backward<kBfloat16>(int shape, unsigned grid, const BackwardArgs &a, hipStream_t stream);

#ifdef CCGLIB_LINEAR_TYPE
template <>
hipError_t launch_backward<CCGLIB_LINEAR_TYPE>(int shape, unsigned grid, const BackwardArgs &a, hipStream_t stream) {
  switch (shape) {
#define CCGLIB_CASE(ID, BX, BY, WX, WY, SLOTS, EU)                                                                 \
  case ID:                                                                                                         \
    if constexpr (backward_in_one(ID)) {                                                                           \
      gemm_linear_backward<CCGLIB_LINEAR_TYPE, BX, BY, WX, WY, SLOTS, EU><<<grid, 64 * WX * WY, 0, stream>>>(a);   \
    }                                                                                                              \
    break;
    CCGLIB_LINEAR_SHAPES(CCGLIB_CASE)
#undef CCGLIB_CASE
  }
  return hipGetLastError();
}
#endif

}  // namespace linear
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_LINEAR_BACKWARD_H_
