// y = act(x W^T + bias) + residual for a few rows of x: single tokens, and experts that have a row or two each.
//
// Bound by memory: W is read once. A block has 16 rows of W and 16 of x; its waves share K out among themselves, CHUNKS x 32
// values at a time each, and are added up at the end, in their order, through LDS. Values go from memory to the registers of the
// 16x16x32 instruction as they are (lane l: 8 values along k of row l % 16), the next ones on their way while the last ones are multiplied:
// no LDS and no barrier in the loop, where gemm_linear's ring waits a round trip a piece. One row of 4096 x 2048: 4.6 us, 9.0 there; of
// 8192 x 8192 out of memory 24.8 (5.4 TB/s), 30.1 there.
#include <algorithm>

#include "linear_gemm.h"

namespace ccglib_amd {
namespace linear {
namespace {

constexpr int kRowsOfW = 16;
// Waves of a block, and 32 values of K of each that are on their way at a time. 4 and 8 against 8 and 4: 16 rows over 64 experts of 2048 x 2048 18.0
// us for 21.6, one row of 8192 x 8192 26.4 for 26.6; half of either: 43 to 50 us for the latter.
constexpr int kRowsWaves = 4, kRowsChunks = 8;

// 8 values of a row from k on; what lies beyond its end (k_all) is zero.
template <bool END> __device__ __forceinline__ int4_t load_8(const char *row, unsigned k, unsigned k_all) {
  if (!END || k + 8 <= k_all) return *reinterpret_cast<const int4_unaligned_t *>(row + (size_t)k * 2);
  int4_t v = {0, 0, 0, 0};
  const unsigned short *const p = reinterpret_cast<const unsigned short *>(row);
#pragma unroll
  for (unsigned e = 0; e < 8; ++e) {
    if (k + e < k_all) v[e / 2] |= (int)((unsigned)p[k + e] << (16 * (e % 2)));
  }
  return v;
}

template <int TYPE> __device__ __forceinline__ float4_t mfma_one(const int4_t &x, const int4_t &y, float4_t c) {
  if constexpr (TYPE == kBfloat16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8_t, x), __builtin_bit_cast(bfloat8_t, y), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(real::half8_t, x), __builtin_bit_cast(real::half8_t, y), c, 0, 0, 0);
  }
}

template <int TYPE, int WAVES, int CHUNKS>
__global__ __launch_bounds__(64 * WAVES) void linear_rows(Args args, StoreParams params) {
  constexpr int BY = kRowsOfX;
  constexpr unsigned STEP = 32 * CHUNKS;
  __shared__ float4_t sums[WAVES][64];
  const int lane = threadIdx.x & 63;
  const unsigned wave = uniform(threadIdx.x >> 6);
  const unsigned fr = lane & 15, g = lane >> 4;
  const unsigned bx = blockIdx.x % args.blocks_x;
  unsigned by = blockIdx.x / args.blocks_x, group = 0;
  Span rows = {0, args.rows};
  if (args.offsets) {
    RowBlocks<BY> blocks(args.offsets, args.groups, args.rows);
    if (by >= blocks.all()) return;
    const RowBlock r = blocks.find(by);
    group = r.group;
    by = r.block;
    rows = r.rows;
  }
  const unsigned x0 = bx * kRowsOfW, y0 = by * BY;
  const unsigned x_row = x0 + fr < args.nx ? x0 + fr : args.nx - 1;      // (rows past the end: never stored)
  const char *const x = args.x + (size_t)group * args.x_group + (size_t)x_row * args.x_pitch;
  const unsigned y_row = y0 + fr < rows.count ? y0 + fr : rows.count - 1;
  const char *const y = args.y + (size_t)(rows.first + y_row) * args.y_pitch;

  float4_t acc = {0.f, 0.f, 0.f, 0.f};
  struct Values {
    int4_t x[CHUNKS], y[CHUNKS];
  };
  auto load = [&](Values &v, unsigned k) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      v.x[c] = load_8<false>(x, k + c * 32 + g * 8, args.k);
      v.y[c] = load_8<false>(y, k + c * 32 + g * 8, args.k);
    }
  };
  auto multiply = [&](const Values &v) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) acc = mfma_one<TYPE>(v.x[c], v.y[c], acc);
  };
  // Whole steps of all waves, then what is left. Blocks begin at different ones: rows lie a multiple of the memory channels' stride
  // apart as often as not, and all blocks at one k ask the same few channels (one row, 8192 x 8192 out of memory: 30.7 us all from the first
  // step on, 24.8 like this).
  const unsigned steps = args.k / (STEP * WAVES), whole = steps * STEP * WAVES;
  if (steps > 0) {
    unsigned step = bx % steps;
    auto next = [&]() {
      const unsigned k = (step * WAVES + wave) * STEP;
      step = step + 1 == steps ? 0 : step + 1;
      return k;
    };
    Values a, b;
    load(a, next());
    unsigned i = 1;
    for (; i + 1 < steps; i += 2) {
      load(b, next());
      multiply(a);
      load(a, next());
      multiply(b);
    }
    if (i < steps) {
      load(b, next());
      multiply(a);
      multiply(b);
    } else {
      multiply(a);
    }
  }
  // What is left, less than a step of all waves: its whole 32 values, two neighbours (a line of the cache) to a wave in turn, and those of the end. All on
  // their way together too (one row, 4096 x 1000: 4.4 us one after the other, 3.7 like this; 8192 x 8000: 23.1 and 22.4).
  const unsigned left_chunks = (args.k - whole) / 32, end = whole + left_chunks * 32;
  const bool has_end = end < args.k && wave == left_chunks / 2 % WAVES;
  int4_t x_end = {0, 0, 0, 0}, y_end = {0, 0, 0, 0};
  if (has_end) {
    x_end = load_8<true>(x, end + g * 8, args.k);
    y_end = load_8<true>(y, end + g * 8, args.k);
  }
  if (wave * 2 < left_chunks) {
    Values v;
#pragma unroll
    for (unsigned c = 0; c < (unsigned)CHUNKS; ++c) {
      const unsigned n = (c / 2 * WAVES + wave) * 2 + c % 2;
      if (n >= left_chunks) break;
      v.x[c] = load_8<false>(x, whole + n * 32 + g * 8, args.k);
      v.y[c] = load_8<false>(y, whole + n * 32 + g * 8, args.k);
    }
#pragma unroll
    for (unsigned c = 0; c < (unsigned)CHUNKS; ++c) {
      if ((c / 2 * WAVES + wave) * 2 + c % 2 < left_chunks) acc = mfma_one<TYPE>(v.x[c], v.y[c], acc);
    }
  }
  if (has_end) acc = mfma_one<TYPE>(x_end, y_end, acc);

  sums[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
  float v[4] = {};
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += sums[w][lane][e];
  }
  const unsigned out_x = x0 + g * 4, left = out_x < args.nx ? args.nx - out_x : 0, row = y0 + fr;
  if (left == 0 || row >= rows.count) return;
  float bias[4] = {};
  if (params.bias) load_row(reinterpret_cast<const typename Value<TYPE>::type *>(params.bias) + (size_t)group * args.nx + out_x, left, bias);
  store_sums<TYPE, kOutput, false>(params, bias, group, rows.first + row, out_x, left, v);
}

}  // namespace

size_t linear_rows_blocks(size_t n) { return ceil_div(n, (size_t)kRowsOfW); }

hipError_t launch_linear_rows(int type, unsigned grid, const Args &a, const StoreParams &s, hipStream_t stream) {
  if (type == kFloat16) {
    linear_rows<kFloat16, kRowsWaves, kRowsChunks><<<grid, 64 * kRowsWaves, 0, stream>>>(a, s);
  } else {
    linear_rows<kBfloat16, kRowsWaves, kRowsChunks><<<grid, 64 * kRowsWaves, 0, stream>>>(a, s);
  }
  return hipGetLastError();
}

}  // namespace linear
}  // namespace ccglib_amd
