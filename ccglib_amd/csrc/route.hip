// Route: for each of T rows of E logits the k largest (ties: the lower number first), their weights by a softmax, and where the T k
// rows lie when they are sorted by expert, those of an expert in their order: an expert's first place plus the number of earlier
// rows that chose it. Two launches: the first chooses, and counts for each tile of rows how many chose which expert; in the second every
// block adds up the tiles before its own and numbers its rows. One tile: one launch. Counts are sums of whole numbers, so that places do not depend
// on the order of blocks.
//
// A row is held by 16 lanes (64 from 257 experts on), PER neighbouring logits a lane, as whole numbers of the same order; each
// round takes the maximum of all lanes by DPP, and the lane that holds it removes it, stores its number and counts it. 16-bit logits have room for their
// number beside them: nothing is removed, a round looks for the largest below the last one.
//
// 65536 rows of 128 float32 logits, 8 chosen of each: 19.7 us to choose (8 rounds of 47 vector instructions for 4 rows a wave, 1.8 us
// each; 6 us would be reading the logits; of bfloat16 12.6, 19 instructions a round for 19.4 us with the other way), 7.5 to place (13 while every block read the tiles' counts as 32 bits and in the same order,
// lines of one channel at a time), 14.6 for the backward pass, which is bound by memory (67 MB, 4.6 TB/s).
#include <algorithm>

#include "linear_gemm.h"
#include "route.h"

namespace ccglib_amd {
namespace {

using linear::Value;

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// Whole numbers in the order of the floats: the two zeros alike, NaN above all, 0 below all.
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned u = v == 0.f ? 0u : __builtin_bit_cast(unsigned, v);
  return v != v ? 0xffffffffu : u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
  if (key == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key);
}

// A 16-bit value's order and, below it, its place among the logits, the first ones highest: no two are alike, so that one maximum says which logit
// it is. 0 is below all.
template <typename T> __device__ __forceinline__ unsigned placed_key_of(float v, unsigned place) {
  const T narrow = (T)v;      // (exact: it was one)
  const unsigned u = v == 0.f ? 0u : __builtin_bit_cast(unsigned short, narrow);
  const unsigned key = v != v ? 0xffffu : u >> 15 ? ~u & 0xffffu : u | 0x8000u;
  return key << 16 | (0xffffu - place);
}
template <typename T> __device__ __forceinline__ float placed_value_of(unsigned key) {
  const unsigned u = key >> 31 ? key >> 16 & 0x7fffu : ~key >> 16;
  return (float)__builtin_bit_cast(T, (unsigned short)u);
}

// What `join` makes of the values of all LANES (16, a DPP row, or 64) that hold a row, in each of them.
template <int LANES, typename T, typename Join> __device__ __forceinline__ T over_lanes(T v, Join join) {
  auto rotated = [&](auto control) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(control)::value, 0xf, 0xf, false));
  };
  v = join(v, rotated(std::integral_constant<int, 0x121>{}));   // row_ror by 1, 2, 4 and 8
  v = join(v, rotated(std::integral_constant<int, 0x122>{}));
  v = join(v, rotated(std::integral_constant<int, 0x124>{}));
  v = join(v, rotated(std::integral_constant<int, 0x128>{}));
  if constexpr (LANES == 64) {
    v = join(v, __shfl_xor(v, 16));
    v = join(v, __shfl_xor(v, 32));
  }
  return v;
}
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ float sum(float a, float b) { return a + b; }

// PER neighbouring logits of a row from `first` on, as floats; `e` logits in all.
template <typename T, int PER> __device__ __forceinline__ void load_logits(const T *row, unsigned first, unsigned e, float (&v)[PER]) {
  linear::load_row(row + first, first < e ? e - first : 0, v);
}

struct ChooseArgs {
  const char *logits;
  int *experts;
  float *weights;
  int *offsets, *slots;
  unsigned short *counts;
  unsigned tokens, e, k, tile, tiles;
  int normalize;
};

// Counts of a tile, 16 bits each: an expert is counted once a row, and no tile has more than kMostRows. Whole quads.
constexpr size_t kMostRows = 65472;
__host__ __device__ __forceinline__ unsigned count_pitch(unsigned experts) { return (experts + 3) / 4 * 4; }

// How many rows of a tile chose an expert, as numbers of the whole array: sums over the tiles before it.
struct Shared {
  unsigned base[kMostExperts];              // an expert's next place
  unsigned below[kMostExperts];
  unsigned waves[kWaves][kMostExperts];
  unsigned totals[kWaves];
};

// First places of all experts from their totals in s.base: sums of what lies in front. All kThreads threads.
__device__ __forceinline__ void first_places(Shared &s, unsigned e) {
  const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const unsigned mine = t < e ? s.base[t] : 0;
  unsigned n = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned other = (unsigned)__shfl_up((int)n, d);
    if (lane >= (unsigned)d) n += other;
  }
  if (lane == 63) s.totals[wave] = n;
  __syncthreads();
  unsigned before = 0;
  for (unsigned w = 0; w < wave; ++w) before += s.totals[w];
  if (t < e) s.base[t] = before + n - mine;
  __syncthreads();
}

// How many lanes below this one have the same expert as it (rank), and how many have it in all; lanes with `have` count.
struct Alike {
  unsigned rank, all;
};
__device__ __forceinline__ Alike alike(bool have, unsigned expert, unsigned e) {
  unsigned long long same = __ballot(have);
  for (unsigned bit = 1; bit < e; bit <<= 1) {
    const unsigned long long set = __ballot((expert & bit) != 0);
    same &= expert & bit ? set : ~set;
  }
  return {(unsigned)__popcll(same & ((1ull << (threadIdx.x & 63)) - 1)), (unsigned)__popcll(same)};
}

// Places of the rows of one tile, `count` of them, from the experts' next places in s.base. Each wave has a piece of them: it counts them,
// learns from the counts of the waves before it where its own begin, and numbers them, 64 at a time. The first 64 kHeld of its
// experts are in registers, loaded long before.
constexpr int kHeld = 4;
struct Piece {
  unsigned from, until;      // rows of the wave
  unsigned held[kHeld];
  __device__ __forceinline__ Piece(const int *experts, unsigned count) {
    const unsigned piece = (count + kThreads - 1) / kThreads * 64;
    from = (threadIdx.x >> 6) * piece;
    until = from + piece < count ? from + piece : count;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const unsigned at = from + h * 64 + (threadIdx.x & 63);
      held[h] = at < until ? (unsigned)experts[at] : 0;
    }
  }
};
__device__ __forceinline__ void place_rows(Shared &s, const Piece &p, const int *experts, int *slots, unsigned e) {
  const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (unsigned i = t; i < e; i += kThreads) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s.waves[w][i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (p.from + h * 64 + lane < p.until) atomicAdd(&s.waves[wave][p.held[h]], 1u);
  }
  for (unsigned at = p.from + kHeld * 64 + lane; at < p.until; at += 64) atomicAdd(&s.waves[wave][experts[at]], 1u);
  __syncthreads();
  for (unsigned i = t; i < e; i += kThreads) {
    unsigned next = s.base[i];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const unsigned n = s.waves[w][i];
      s.waves[w][i] = next;
      next += n;
    }
  }
  __syncthreads();
  auto number = [&](unsigned at, unsigned mine) {
    const bool have = at + lane < p.until;
    const Alike a = alike(have, mine, e);
    const unsigned place = s.waves[wave][mine] + a.rank;
    if (have) slots[at + lane] = (int)place;
    __builtin_amdgcn_wave_barrier();       // (all lanes have read, before the first of each expert writes)
    if (have && a.rank == 0) s.waves[wave][mine] = place + a.all;
    __builtin_amdgcn_wave_barrier();
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (p.from + h * 64 < p.until) number(p.from + h * 64, p.held[h]);
  }
  for (unsigned at = p.from + kHeld * 64; at < p.until; at += 64) number(at, at + lane < p.until ? (unsigned)experts[at + lane] : 0);
}

template <int TYPE, int LANES, int PER> __global__ __launch_bounds__(kThreads) void route_choose(ChooseArgs a) {
  using T = typename Value<TYPE>::type;
  __shared__ Shared s;
  for (unsigned i = threadIdx.x; i < a.e; i += kThreads) s.base[i] = 0;
  __syncthreads();
  const unsigned group = threadIdx.x / LANES, l = threadIdx.x % LANES;
  const unsigned begin = blockIdx.x * a.tile, end = a.tokens - begin < a.tile ? a.tokens : begin + a.tile;
  float ahead[PER];      // the next row's logits, on their way
  if (begin + group < end) load_logits(reinterpret_cast<const T *>(a.logits) + (size_t)(begin + group) * a.e, l * PER, a.e, ahead);
  for (unsigned t = begin + group; t < end; t += kThreads / LANES) {
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = ahead[i];
    const unsigned next = t + kThreads / LANES;
    if (next < end) load_logits(reinterpret_cast<const T *>(a.logits) + (size_t)next * a.e, l * PER, a.e, ahead);
    unsigned keys[PER];
    const size_t at = (size_t)t * a.k;
    float top, my_value;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < PER; ++i) keys[i] = l * PER + i < a.e ? placed_key_of<T>(v[i], l * PER + i) : 0u;
      unsigned my_key = 0, top_key = 0, last = 0;
      for (unsigned j = 0; j < a.k; ++j) {
        // the largest below the last one: of the differences from it, modulo 2^32, those of the keys that have been taken are the smallest
        unsigned best = keys[0] - last;
#pragma unroll
        for (int i = 1; i < PER; ++i) best = larger(best, keys[i] - last);
        last += over_lanes<LANES>(best, larger);
        if (j == 0) top_key = last;
        my_key = l == j ? last : my_key;
      }
      top = placed_value_of<T>(top_key);
      my_value = placed_value_of<T>(my_key);
      if (l < a.k) {
        const unsigned number = 0xffffu - (my_key & 0xffffu);
        a.experts[at + l] = (int)number;
        atomicAdd(&s.base[number], 1u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) keys[i] = l * PER + i < a.e ? key_of(v[i]) : 0u;
      unsigned my_key = 0, top_key = 0;
      for (unsigned j = 0; j < a.k; ++j) {
        unsigned best = keys[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = larger(best, keys[i]);
        const unsigned most = over_lanes<LANES>(best, larger);
        // the lowest lane of the row that holds it, and its lowest logit that does
        const unsigned long long holders = __ballot(best == most) >> (threadIdx.x & 63 & ~(LANES - 1));
        const bool winner = l == (unsigned)__builtin_ctzll(holders);
        bool open = winner;
        unsigned number = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const bool hit = open && keys[i] == most;
          open = open && !hit;
          keys[i] = hit ? 0u : keys[i];
          number = hit ? i : number;
        }
        if (winner) {
          number += l * PER;
          a.experts[at + j] = (int)number;
          atomicAdd(&s.base[number], 1u);
        }
        if (j == 0) top_key = most;
        my_key = l == j ? most : my_key;
      }
      top = value_of(top_key);
      my_value = value_of(my_key);
    }
    // (a row of nothing but -inf has weights of zero)
    const float over = top == -__builtin_inff() ? 0.f : top;
    const float mine = l < a.k ? __expf(my_value - over) : 0.f;
    float all;
    if (a.normalize) {
      all = over_lanes<LANES>(mine, sum);
    } else {
      float some = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) some += l * PER + i < a.e ? __expf(v[i] - over) : 0.f;
      all = over_lanes<LANES>(some, sum);
    }
    if (l < a.k) {
      a.weights[at + l] = all == 0.f ? 0.f : mine / all;
    }
  }
  __syncthreads();
  if (a.tiles > 1) {
    const unsigned pitch = count_pitch(a.e);
    for (unsigned i = threadIdx.x; i < pitch; i += kThreads) {
      a.counts[(size_t)blockIdx.x * pitch + i] = i < a.e ? (unsigned short)s.base[i] : 0;
    }
    return;
  }
  first_places(s, a.e);
  for (unsigned i = threadIdx.x; i < a.e; i += kThreads) a.offsets[i] = (int)s.base[i];
  if (threadIdx.x == 0) a.offsets[a.e] = (int)(a.tokens * a.k);
  __syncthreads();       // (the block's own stores of a.experts are behind the barrier before)
  place_rows(s, Piece(a.experts, a.tokens * a.k), a.experts, a.slots, a.e);
}

__global__ __launch_bounds__(kThreads) void route_place(ChooseArgs a) {
  __shared__ Shared s;
  const unsigned t = threadIdx.x;
  const unsigned begin = blockIdx.x * a.tile, end = a.tokens - begin < a.tile ? a.tokens : begin + a.tile;
  const int *const experts = a.experts + (size_t)begin * a.k;
  const Piece piece(experts, (end - begin) * a.k);
  // A thread adds up four experts of every so many tiles: its loads are on their way together. Each block begins at its own tile: if
  // all read the same lines at the same time, one channel of the cache has them all to itself.
  const unsigned quads = count_pitch(a.e) / 4, ways = kThreads / quads, quad = t % quads, way = t / quads;
  unsigned all[4] = {}, below[4] = {};
  if (way < ways) {
#pragma unroll 8
    for (unsigned i = way; i < a.tiles; i += ways) {
      const unsigned b = i + blockIdx.x < a.tiles ? i + blockIdx.x : i + blockIdx.x - a.tiles;
      const uint2 n = reinterpret_cast<const uint2 *>(a.counts)[(size_t)b * quads + quad];
      const unsigned each[4] = {n.x & 0xffff, n.x >> 16, n.y & 0xffff, n.y >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        all[j] += each[j];
        below[j] += b < blockIdx.x ? each[j] : 0;
      }
    }
  }
  for (unsigned i = t; i < count_pitch(a.e); i += kThreads) s.base[i] = s.below[i] = 0;
  __syncthreads();
  if (way < ways) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      atomicAdd(&s.base[quad * 4 + j], all[j]);
      atomicAdd(&s.below[quad * 4 + j], below[j]);
    }
  }
  __syncthreads();
  first_places(s, a.e);
  if (blockIdx.x == 0) {
    for (unsigned i = t; i < a.e; i += kThreads) a.offsets[i] = (int)s.base[i];
    if (t == 0) a.offsets[a.e] = (int)(a.tokens * a.k);
  }
  for (unsigned i = t; i < a.e; i += kThreads) s.base[i] += s.below[i];
  place_rows(s, piece, experts, a.slots + (size_t)begin * a.k, a.e);      // (begins with a barrier)
}

struct BackwardArgs {
  const char *logits;
  const int *experts;
  const float *weights, *dweights;
  char *dlogits;
  unsigned tokens, e, k;
  int normalize;
};

// inner = sum_j w_j dw_j;  normalized: dl_e = w_j (dw_j - inner) at the chosen, 0 elsewhere (the softmax is one of the chosen);
// else dl_e = p_e ((dw_j at the chosen, 0 elsewhere) - inner). Bound by memory.
template <int TYPE, int LANES, int PER> __global__ __launch_bounds__(256) void route_backward(BackwardArgs a) {
  using T = typename Value<TYPE>::type;
  const unsigned l = threadIdx.x % LANES, t = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (t >= a.tokens) return;      // (all lanes of a row together)
  const size_t at = (size_t)t * a.k + l;
  const unsigned expert = l < a.k ? (unsigned)a.experts[at] : 0xffffffffu;
  const float w = l < a.k ? a.weights[at] : 0.f, dw = l < a.k ? a.dweights[at] : 0.f;
  const float inner = over_lanes<LANES>(w * dw, sum);
  float d[PER] = {}, p[PER];
  if (!a.normalize) {
    load_logits(reinterpret_cast<const T *>(a.logits) + (size_t)t * a.e, l * PER, a.e, p);
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (l * PER + i >= a.e) p[i] = -__builtin_inff();
      top = p[i] > top || p[i] != p[i] ? p[i] : top;
    }
    top = over_lanes<LANES>(top, [](float x, float y) { return x != x || x > y ? x : y; });
    const float over = top == -__builtin_inff() ? 0.f : top;
    float some = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      p[i] = __expf(p[i] - over);
      some += p[i];
    }
    const float all = over_lanes<LANES>(some, sum), scale = all == 0.f ? 0.f : 1.f / all;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      p[i] *= scale;
      d[i] = -inner;
    }
  }
  const float mine = a.normalize ? w * (dw - inner) : dw;
  for (unsigned j = 0; j < a.k; ++j) {
    const int from = (int)((threadIdx.x & 63) / LANES * LANES + j);
    const unsigned chosen = (unsigned)__shfl((int)expert, from);
    const float add = __shfl(mine, from);
#pragma unroll
    for (int i = 0; i < PER; ++i) d[i] += l * PER + i == chosen ? add : 0.f;
  }
  if (!a.normalize) {
#pragma unroll
    for (int i = 0; i < PER; ++i) d[i] *= p[i];
  }
  if (l * PER < a.e) real::store_row(reinterpret_cast<T *>(a.dlogits) + (size_t)t * a.e + l * PER, a.e - l * PER, d);
}

// Calls `f` with the lanes of a row and the logits of a lane.
template <typename F> void by_experts(unsigned e, F &&f) {
  using std::integral_constant;
  if (e <= 16) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if (e <= 32) return f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  if (e <= 64) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  if (e <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  if (e <= 256) return f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  if (e <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
  return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}
template <typename F> void by_type(int type, F &&f) {
  using std::integral_constant;
  if (type == kFloat32) return f(integral_constant<int, kFloat32>{});
  if (type == kFloat16) return f(integral_constant<int, kFloat16>{});
  return f(integral_constant<int, kBfloat16>{});
}

}  // namespace

void plan_route(RouteParams *p) {
  // 256 tiles where counts of 16 bits allow it: each block adds up the counts of all
  const size_t least = 64;
  p->tile = (unsigned)std::min(kMostRows, std::max(least, ceil_div(ceil_div(p->tokens, (size_t)256), least) * least));
  p->tiles = (unsigned)std::max<size_t>(1, ceil_div(p->tokens, (size_t)p->tile));
}

size_t route_workspace_bytes(const RouteParams &p) { return p.tiles > 1 ? sizeof(unsigned short) * p.tiles * count_pitch(p.experts) : 0; }

hipError_t launch_route(const RouteParams &p, const void *logits, int *experts, float *weights, int *offsets, int *slots,
                        hipStream_t stream) {
  const ChooseArgs a = {static_cast<const char *>(logits), experts, weights, offsets, slots, p.counts, p.tokens, p.experts,
                        p.chosen, p.tile, p.tiles, p.normalize};
  by_type(p.type, [&](auto type) {
    by_experts(p.experts, [&](auto lanes, auto per) {
      route_choose<decltype(type)::value, decltype(lanes)::value, decltype(per)::value><<<p.tiles, kThreads, 0, stream>>>(a);
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.tiles == 1) return e;
  route_place<<<p.tiles, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_route_backward(const RouteParams &p, const void *logits, const int *experts, const float *weights,
                                 const float *dweights, void *dlogits, hipStream_t stream) {
  if (p.tokens == 0) return hipSuccess;
  const BackwardArgs a = {static_cast<const char *>(logits), experts, weights, dweights, static_cast<char *>(dlogits), p.tokens,
                          p.experts, p.chosen, p.normalize};
  by_type(p.type, [&](auto type) {
    by_experts(p.experts, [&](auto lanes, auto per) {
      const unsigned grid = (unsigned)ceil_div(p.tokens, (size_t)(256 / decltype(lanes)::value));
      route_backward<decltype(type)::value, decltype(lanes)::value, decltype(per)::value><<<grid, 256, 0, stream>>>(a);
    });
  });
  return hipGetLastError();
}

}  // namespace ccglib_amd
