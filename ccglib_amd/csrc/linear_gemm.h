// Products of 16-bit values for linear layers, on the matrix cores:
//   D[y][x] = sum_k X[x][k] Y[y][k],   x the contiguous axis of D,
// where each operand lies as it is, rows along k or rows along its own index, so that the three products of a layer
// read x [M][K], W [N][K] and dz [M][N] in place:
//   kOutput   y = x W^T     X = W, Y = x, both with k contiguous
//   kInput     dx = dz W     X = W, whose rows run along x here; Y = dz with k (the layer's outputs) contiguous
//   kWeights   dW = dz^T x   X = x, Y = dz, k the rows of both
// Rows may belong to groups (experts), offsets[g] to offsets[g + 1] - 1 to group g, each with a W of its own: D's rows
// of a group are multiplied with that W, or (kWeights) k runs over the group's rows and D is the group's.
//
// K is walked in pieces of 64 values. LDS holds a ring of SLOTS pieces; copies go straight there (1 KiB an instruction).
//   k contiguous: rows of 128 bytes, chunk c (16 bytes) of row r at c ^ (r & 7); a lane reads its 8 values at once.
//   k strided: 64 rows of k, the block's columns of each; a 16x16x32 fragment, which wants 8 values along k in a lane,
//   is read by ds_read_b64_tr_b16, which transposes 4 x 16 values inside 16 lanes. Pieces of the columns are XORed with
//   bits of k, so that the 4 rows that 16 lanes read lie in different banks. 32 lanes read at a time: those of Y, and of X in pieces of 32 bytes
//   (192 columns), all in different banks; those of X in pieces of 64 bytes, of which a read takes half, two in each of 32 banks.
// X supplies the instruction's rows, in an order that leaves a lane with 4 NT neighbours in x: wide stores.
//
// Ends. Rows beyond an operand are clamped (their sums are never stored), k beyond the end reads zeros. Where a row along k
// does not end with a chunk, its last chunk is read 8 values before the end, and the values that the chunk before
// it has already brought are zeroed in registers, in the last piece; where the other operand's k is strided, its rows are
// taken in the same order. The one access that could leave the memory of an operand, the chunk at its very end,
// is read from a copy (x_tail, y_tail: see Tail).
//
// What bounds it. 8192^3 takes 765 to 805 us in each of the three products (1370 to 1440 TFLOP/s): matrix instructions are busy 67 % of the cycles, at
// 1.95 to 2.0 GHz; without its copies it would be 646, without the barrier 749. A wave's 128 x 64 of a 256 x 256 block read 96 bytes of LDS
// a cycle of matrix instructions and unit, of 128 that there are; 64 x 64 of the smaller blocks would read 128, which is why they are only for what 256 x 256 leaves
// idle. In dx and dW X's reads take twice their time (40 % of LDS's busy cycles, which are 1.7 times y's), as 160 bytes would: 107 a cycle at 67 %. A
// block's start and stores take 9 us (12 with an activation) of a round that multiplies 1.5 us a piece: one block a unit, nothing
// runs beside them. Two blocks of 256 x 128 a unit, in pieces of 32 values, hide them and are slower all the same (8192^3 992; 4096 rows over 32
// experts of 1024 x 2048 38 for 35).
#ifndef CCGLIB_AMD_LINEAR_GEMM_H_
#define CCGLIB_AMD_LINEAR_GEMM_H_

#include "linear.h"
#include "real_gemm.h"

namespace ccglib_amd {
namespace linear {

using real::float4_t;
using real::Fragment;
using real::pin;
using real::static_for;
using real::uniform;

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bfloat8_t __attribute__((ext_vector_type(8)));

constexpr int kPiece = 64;   // values of K

// The end of an operand's memory, and a copy of its last 16 values with 8 zeros behind them: a chunk that starts less than 16 bytes before
// `end` is read from there. copy null: no chunk leaves the operand.
struct Tail {
  const char *copy, *end;
};

struct Args {
  const char *x, *y;
  unsigned nx, ny, k;
  unsigned x_pitch, y_pitch;       // bytes from row to row
  Tail x_tail, y_tail;
  const int *offsets;              // of groups; null: one, with all rows
  unsigned groups, rows;           // offsets count to `rows` at most
  size_t x_group;                  // bytes from one group's X to the next (kOutput, kInput)
  unsigned blocks_x, blocks_y;     // (of a group: kWeights)
  unsigned parts, pieces_per_part; // as in real_gemm.h
  unsigned rotate;                 // blocks begin at different pieces of K (see below)
  float *partial;
  unsigned *arrived;
};

// Where group g's rows are: [first, first + count). Whatever the offsets hold, this lies inside the `rows` there are.
struct Span {
  unsigned first, count;
};
__device__ __forceinline__ Span span_of(const int *offsets, unsigned g, unsigned rows) {
  const int a = offsets[g], b = offsets[g + 1];
  Span s;
  s.first = a < 0 ? 0u : (unsigned)a > rows ? rows : (unsigned)a;
  const unsigned end = b < 0 ? 0u : (unsigned)b > rows ? rows : (unsigned)b;
  s.count = end > s.first ? end - s.first : 0u;
  return s;
}

// Groups' blocks of BY rows, numbered one after the other. Each wave looks for itself, 64 groups at a time, a lane each.
struct RowBlock {
  unsigned group, block;    // which group, and which of its blocks
  Span rows;                // the group's
};
template <int BY> class RowBlocks {
 public:
  __device__ __forceinline__ RowBlocks(const int *offsets, unsigned groups, unsigned rows)
      : offsets_(offsets), groups_(groups), rows_(rows) {
    load(0);
    all_ = last_lane(until_);
    if (groups > 64) {
      for (unsigned g = 64; g < groups; g += 64) {
        load(g);
        all_ += last_lane(until_);
      }
    }
  }
  __device__ __forceinline__ unsigned all() const { return all_; }
  // Block `target` of all() (which is less).
  __device__ __forceinline__ RowBlock find(unsigned target) {
    unsigned from = 0;
    if (groups_ > 64) {
      for (;; from += 64) {
        load(from);
        const unsigned here = last_lane(until_);
        if (target < here || from + 64 >= groups_) break;
        target -= here;
      }
    }
    const unsigned long long behind = __ballot(until_ > target);
    const int lane = behind ? __builtin_ctzll(behind) : 63;
    RowBlock r;
    r.group = uniform(from + lane);
    r.rows.first = (unsigned)__builtin_amdgcn_readlane((int)mine_.first, lane);
    r.rows.count = (unsigned)__builtin_amdgcn_readlane((int)mine_.count, lane);
    r.block = target - ((unsigned)__builtin_amdgcn_readlane((int)until_, lane) - (r.rows.count + BY - 1) / BY);
    return r;
  }

 private:
  static __device__ __forceinline__ unsigned last_lane(unsigned v) { return (unsigned)__builtin_amdgcn_readlane((int)v, 63); }
  // until_: blocks of this lane's group and those of lower lanes
  __device__ __forceinline__ void load(unsigned from) {
    const unsigned lane = threadIdx.x & 63, g = from + lane;
    mine_ = {0, 0};
    if (g < groups_) mine_ = span_of(offsets_, g, rows_);
    until_ = (mine_.count + BY - 1) / BY;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned other = (unsigned)__shfl_up((int)until_, d);
      if (lane >= (unsigned)d) until_ += other;
    }
  }
  const int *offsets_;
  unsigned groups_, rows_, all_, until_;
  Span mine_;
};

// The group that is `nth` if those with many rows go first, in five classes of their number: dW's blocks take as long as their group's rows are many, and
// a long one that begins last keeps the others waiting (us, as they come and like this: 16384 rows, up to 3224 of a group, over 8 of 2048 x 2048
// 149 and 133; 4096, up to 395, over 32 of 1024 x 2048 73 and 68; 8192, up to 585, over 64 of 2048 x 1024 163 and 151; of 15 such cases the
// mean is 0.97, the worst 1.02). Beyond 64 groups each of them is a small part of the whole: as they come.
__device__ __forceinline__ unsigned by_length(const Args &a, unsigned nth) {
  if (a.groups > 64) return nth;
  const unsigned lane = threadIdx.x & 63;
  const bool have = lane < a.groups;
  const float times = have ? (float)span_of(a.offsets, lane, a.rows).count * (float)a.groups / (float)a.rows : 0.f;   // the mean's
  const int mine = times >= 4.f ? 0 : times >= 2.f ? 1 : times >= 1.f ? 2 : times >= 0.5f ? 3 : 4;
  unsigned long long these = 0;
  for (int c = 0; c < 5; ++c) {
    these = __ballot(have && mine == c);
    const unsigned n = (unsigned)__popcll(these);
    if (nth < n) break;
    nth -= n;
  }
  for (; nth > 0; --nth) these &= these - 1;
  return uniform((unsigned)__builtin_ctzll(these));
}

// Which part of D a workgroup has.
struct Place {
  bool none;
  unsigned group, bx, by, part, tile;
  Span rows;                // the group's
  unsigned cut, piece;      // the workgroup has one of `cut` pieces of the block
};

// Blocks of the last round, where they are so few that the units hold two or four pieces of each of them: how many, and what they are
// cut into (gemm_linear_cut).
constexpr unsigned kUnits = 256;
struct LastRound {
  unsigned blocks, cut;
};
__host__ __device__ __forceinline__ LastRound last_round(unsigned blocks) {
  const unsigned rest = blocks % kUnits;
  return {rest, rest > kUnits / 2 ? 1u : rest > kUnits / 4 ? 2u : 4u};
}
// More workgroups than blocks, at most
constexpr unsigned kMostCut = 3 * kUnits / 4;

// Block `id` of `count` that a launch has for the product. CUT: the last round's blocks are cut.
template <int KIND, int BY, bool CUT> __device__ __forceinline__ Place place(const Args &a, unsigned id, unsigned count) {
  Place p;
  p.none = false;
  p.group = p.part = p.piece = 0;
  p.cut = 1;
  p.rows = {0, a.rows};
  // groups of four block rows, y fastest: the blocks that an XCD works on at one time share rows of X and of Y
  auto spread = [&](unsigned t, unsigned blocks_y) {
    constexpr unsigned GROUP = 4;
    const unsigned g = t / (GROUP * a.blocks_x), in = t - g * GROUP * a.blocks_x;
    const unsigned rows = blocks_y - g * GROUP < GROUP ? blocks_y - g * GROUP : GROUP;
    p.by = uniform(g * GROUP + in % rows);
    p.bx = uniform(in / rows);
    p.tile = uniform(t);
  };
  // Which of all blocks, in the order of the XCDs
  auto order = [&](unsigned all) {
    if constexpr (CUT) {
      const LastRound last = last_round(all);
      const unsigned whole = all - last.blocks;
      if (id >= whole) {
        if (id - whole >= last.blocks * last.cut) return all;
        const unsigned n = xcd_remap(id - whole, last.blocks * last.cut);
        p.cut = uniform(last.cut);
        p.piece = uniform(n % last.cut);
        return whole + n / last.cut;
      }
      return xcd_remap(id, whole);
    }
    return id < all ? xcd_remap(id, all) : all;
  };
  if (a.offsets && KIND != kWeights) {
    RowBlocks<BY> blocks(a.offsets, a.groups, a.rows);
    const unsigned all = blocks.all() * a.blocks_x;
    const unsigned t = order(all);
    if (t >= all) {
      p.none = true;
      return p;
    }
    spread(t, blocks.all());
    const RowBlock r = blocks.find(p.by);
    p.group = r.group;
    p.by = r.block;
    p.rows = r.rows;
    return p;
  }
  const unsigned per_matrix = a.blocks_x * a.blocks_y;
  if (a.offsets) {
    // (each XCD has an eighth of every group's blocks: groups differ in their rows)
    const unsigned nth = uniform(id / per_matrix);
    p.group = by_length(a, nth);
    spread(xcd_remap(id - nth * per_matrix, per_matrix), a.blocks_y);
    p.rows = span_of(a.offsets, p.group, a.rows);
    p.rows.first = uniform(p.rows.first);
    p.rows.count = uniform(p.rows.count);
  } else {
    const unsigned t = order(CUT ? per_matrix : count);
    p.part = uniform(t / per_matrix);
    spread(t - p.part * per_matrix, a.blocks_y);
  }
  return p;
}

// Bits of k that the number of a unit (32 or 64 bytes of columns) is XORed with, for rows of ROW bytes: the 4 rows that 16 lanes read
// start in different banks (256 bytes of them). The next 16 lanes' 4, in steps of 8, lie in the other banks with units of 32 bytes; with units
// of 64 they lie in the same ones, two ways: a read takes 8 of each 16 bytes, and so half of the banks whatever the order of units.
template <int ROW, int UNIT> __device__ __forceinline__ unsigned unit_swizzle(unsigned k) {
  if constexpr (ROW % 256 == 0) return UNIT == 32 ? (k & 3) | (k >> 3 & 1) << 2 : k & 3;
  if constexpr (ROW % 128 == 0) return UNIT == 32 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : k >> 1 & 1;
  return UNIT == 32 ? k >> 3 & 1 : 0;
}

template <int TYPE> __device__ __forceinline__ float4_t mfma(const Fragment &x, const Fragment &y, float4_t c, int q) {
  const int4_t a = q == 0 ? __builtin_shufflevector(x, x, 0, 1, 2, 3) : __builtin_shufflevector(x, x, 4, 5, 6, 7);
  const int4_t b = q == 0 ? __builtin_shufflevector(y, y, 0, 1, 2, 3) : __builtin_shufflevector(y, y, 4, 5, 6, 7);
  if constexpr (TYPE == kBfloat16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8_t, a), __builtin_bit_cast(bfloat8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(real::half8_t, a), __builtin_bit_cast(real::half8_t, b), c, 0, 0, 0);
  }
}

template <int TYPE> struct Value;
template <> struct Value<kFloat16> { using type = _Float16; };
template <> struct Value<kBfloat16> { using type = __bf16; };
template <> struct Value<kFloat32> { using type = float; };

// 1 / (1 + e^-a)
__device__ __forceinline__ float sigmoid(float a) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a * -1.44269504088896341f));
}
// gelu(z) = z sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3)), which is z/2 (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3)))
constexpr float kGelu1 = 1.59576912160573071f, kGelu3 = 0.071354816272600f;   // 2 sqrt(2/pi), and 0.044715 times that
__device__ __forceinline__ float gelu_argument(float z) { return z * __builtin_fmaf(kGelu3 * z, z, kGelu1); }

template <int N> __device__ __forceinline__ void activate(int activation, float (&v)[N]) {
  if (activation == kRelu) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = v[e] > 0.f ? v[e] : v[e] <= 0.f ? 0.f : v[e];   // (NaN stays)
  } else if (activation == kGelu) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= sigmoid(gelu_argument(v[e]));
  } else if (activation == kSilu) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= sigmoid(v[e]);
  }
}

// N neighbours from `from` on, of which `left` are inside the row, as floats; what lies beyond is zero.
template <typename T, int N> __device__ __forceinline__ void load_row(const T *from, unsigned left, float (&v)[N]) {
  constexpr int E = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
  typedef T piece_t __attribute__((ext_vector_type(E), aligned(sizeof(T))));
  if (left >= (unsigned)N) {
#pragma unroll
    for (int i = 0; i < N; i += E) {
      const piece_t w = *reinterpret_cast<const piece_t *>(from + i);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i + e] = (float)w[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (unsigned)e < left ? (float)from[e] : 0.f;
  }
}

// real::store_row, past the caches: what is more than the last-level cache holds is not in it when it is read next, and only
// displaces operands (8192^3 with residual and z: 874 us in the ordinary way, 827 past).
template <typename T, int N> __device__ __forceinline__ void store_row(bool past, T *to, unsigned left, const float (&v)[N]) {
  constexpr int E = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
  typedef T piece_t __attribute__((ext_vector_type(E)));
  typedef piece_t piece_unaligned_t __attribute__((aligned(sizeof(T))));
  if (past && left >= (unsigned)N) {
#pragma unroll
    for (int i = 0; i < N; i += E) {
      piece_unaligned_t w;
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = (T)v[i + e];
      __builtin_nontemporal_store(w, reinterpret_cast<piece_unaligned_t *>(to + i));
    }
  } else {
    real::store_row(to, left, v);
  }
}

// What becomes of the sums of D.
struct StoreParams {
  char *out, *z;                  // z: may be null (kOutput)
  const char *bias, *residual;    // may be null (kOutput)
  size_t pitch;                   // elements from row to row of out, z and residual
  size_t group;                   // elements from one group's out to the next (kWeights)
  int activation;
  int wide, accumulate;           // kWeights: out is float32, and added to
  int past;                       // out and z are stored past the caches
};

// `v`: N neighbours from x on (`left` of them inside the row) in row y of D, or of all groups' rows. LINES: the wave writes whole cache lines, one
// part right behind the other (parts of lines past the caches: 192 x 192 blocks of 268 MB of dW 301 us, 159 in the ordinary way).
template <int TYPE, int KIND, bool LINES, int N>
__device__ __forceinline__ void store_sums(const StoreParams &p, const float (&bias)[N], unsigned group, unsigned y, unsigned x,
                                           unsigned left, float (&v)[N]) {
  using T = typename Value<TYPE>::type;
  const size_t at = (size_t)y * p.pitch + x;
  if constexpr (KIND == kOutput) {
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += bias[e];
    }
    if (p.z) store_row(LINES && p.past, reinterpret_cast<T *>(p.z) + at, left, v);
    activate(p.activation, v);
    if (p.residual) {
      float r[N];
      load_row(reinterpret_cast<const T *>(p.residual) + at, left, r);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += r[e];
    }
    store_row(LINES && p.past, reinterpret_cast<T *>(p.out) + at, left, v);
  } else if constexpr (KIND == kInput) {
    store_row(LINES && p.past, reinterpret_cast<T *>(p.out) + at, left, v);
  } else {
    const size_t here = (size_t)group * p.group + at;
    if (!p.wide) {
      store_row(LINES && p.past, reinterpret_cast<T *>(p.out) + here, left, v);
    } else {
      float *const out = reinterpret_cast<float *>(p.out) + here;
      if (p.accumulate) {
        float old[N];
        load_row(out, left, old);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += old[e];
      }
      store_row(LINES && p.past, out, left, v);
    }
  }
}

// The same for 32 bits of dW in 32 columns that are all inside, x the first of the lane's first four: lanes 16 apart hold 8 neighbours each, and
// exchange them so that a store writes 64 bytes of a row in one piece, not 16 of each 32. 256 x 256 blocks, us: 512 rows over 16
// experts of 4096 x 4096 472 and 222 (1 GiB), 8192 rows over 64 of 2048 x 1024 213 and 158, 2048 x 8192 x 8192 262 and 235. (Waves
// of 64 columns lose as often as they gain: 32 of 1024 x 2048 78 and 97, 16 of 4096 x 4096 429 and 243, 2048 x 8192 x 8192 272 and 289. Whole lines by one store
// more: nothing gained, and 10 to 20 % lost where old values are added to.)
template <bool LINES>
__device__ __forceinline__ void store_wide(const StoreParams &p, unsigned group, unsigned y, unsigned x, float4_t a, float4_t b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float lower = a[e], upper = b[e];
    const auto rows = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, lower), __builtin_bit_cast(unsigned, upper), false, false);
    const auto halves = __builtin_amdgcn_permlane32_swap(rows[0], rows[1], false, false);
    const unsigned first = halves[0], second = halves[1];
    a[e] = __builtin_bit_cast(float, first);
    b[e] = __builtin_bit_cast(float, second);
  }
  float *const out = reinterpret_cast<float *>(p.out) + (size_t)group * p.group + (size_t)y * p.pitch + x;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[4], old[4] = {};
    if (p.accumulate) load_row(out + h * 16, 4, old);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (h ? b : a)[e] + old[e];
    store_row(LINES && p.past, out + h * 16, 4, v);
  }
}

template <int BX, int BY, int SLOTS> constexpr int kLdsBytes = SLOTS *(BX + BY) * kPiece * 2;

// The block of D from x0, y0 on. lds: kLdsBytes, at a multiple of 256.
template <int TYPE, int KIND, int BX, int BY, int WX, int WY, int SLOTS>
__device__ __forceinline__ void product_at(const Args &args, const StoreParams &params, char *lds, const Place &at, unsigned x0,
                                           unsigned y0) {
  constexpr bool X_ROWS = KIND == kOutput, Y_ROWS = KIND != kWeights;     // k is contiguous
  constexpr int WAVES = WX * WY, TX = BX / WX, TY = BY / WY, NX = TX / 16, NY = TY / 16;
  constexpr int NT = NX % 2 ? 1 : 2, UNIT_X = 32 * NT;
  constexpr int X_BYTES = BX * kPiece * 2, Y_BYTES = BY * kPiece * 2, SLOT_BYTES = X_BYTES + Y_BYTES;
  constexpr int X_COPIES = BX / 8 / WAVES, Y_COPIES = BY / 8 / WAVES, COPIES = X_COPIES + Y_COPIES;
  static_assert(BX / 8 % WAVES == 0 && BY / 8 % WAVES == 0, "a wave's copies are of one operand each");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wx = wave % WX, wy = wave / WX;
  // rows of Y and length of K that this block's group has
  const unsigned ny = Y_ROWS && args.offsets ? at.rows.count : args.ny;
  const unsigned k_all = !Y_ROWS && args.offsets ? at.rows.count : args.k;
  const unsigned pieces = k_all / kPiece + (k_all % kPiece != 0);
  const unsigned first = at.part * args.pieces_per_part;
  const unsigned last = args.parts == 1 || pieces - first < args.pieces_per_part ? pieces : first + args.pieces_per_part;
  const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

  // ---- copies ----
  // Row 0 of k of a group where k is strided, row 0 of the block where it is contiguous
  const char *x_next = args.x, *y_next = args.y;
  if (args.offsets) {
    if constexpr (KIND == kWeights) {
      x_next += (size_t)at.rows.first * args.x_pitch;
    } else {
      x_next += (size_t)at.group * args.x_group;
    }
    y_next += (size_t)at.rows.first * args.y_pitch;
  }
  constexpr unsigned PIECE_BYTES = kPiece * 2;
  x_next += X_ROWS ? (size_t)x0 * args.x_pitch + (size_t)first * PIECE_BYTES : (size_t)x0 * 2 + (size_t)first * kPiece * args.x_pitch;
  y_next += Y_ROWS ? (size_t)y0 * args.y_pitch + (size_t)first * PIECE_BYTES : (size_t)y0 * 2 + (size_t)first * kPiece * args.y_pitch;
  const size_t x_step = X_ROWS ? PIECE_BYTES : (size_t)kPiece * args.x_pitch, y_step = Y_ROWS ? PIECE_BYTES : (size_t)kPiece * args.y_pitch;
  const unsigned chunk = (unsigned)((lane & 7) ^ (lane >> 3));       // (k contiguous: the same in all copies)
  unsigned offset[COPIES];
#pragma unroll
  for (int n = 0; n < COPIES; ++n) {
    const bool of_x = n < X_COPIES;
    const int q = wave + (of_x ? n : n - X_COPIES) * WAVES;
    const unsigned most = (of_x ? args.nx - x0 : ny - y0) - 1, pitch = of_x ? args.x_pitch : args.y_pitch;
    if (of_x ? X_ROWS : Y_ROWS) {
      const int row = q * 8 + (lane >> 3);
      unsigned want = row;
      if (of_x) {   // row `row` of LDS holds this row of the block
        const int in = row % (16 * NT), t = in / 16, r = in % 16;
        want = row - in + (r >> 2) * (4 * NT) + t * 4 + (r & 3);
      }
      offset[n] = (want < most ? want : most) * pitch + chunk * 16;
    } else {
      constexpr int X_CHUNKS = BX / 8, Y_CHUNKS = BY / 8;
      const unsigned place = q * 64 + lane, k = of_x ? place / X_CHUNKS : place / Y_CHUNKS;
      unsigned c = of_x ? place % X_CHUNKS : place % Y_CHUNKS;       // 16 bytes of row k
      if (of_x) {
        constexpr int PER = UNIT_X / 16;
        c = (c / PER ^ unit_swizzle<BX * 2, UNIT_X>(k)) * PER + c % PER;
      } else {
        c = (c / 2 ^ unit_swizzle<BY * 2, 32>(k)) * 2 + c % 2;
      }
      offset[n] = k * pitch + (c * 8 <= most ? c * 16 : 0);
    }
  }
  // (kept in registers: its address is a scalar load, behind which the LDS reads would be waited for all together)
  const char *zeros = real::g_zeros;
  real::pin_scalar(zeros);
  // Blocks whose Y stays in the caches whatever they ask for begin at different pieces of K: rows lie a multiple of the memory
  // channels' stride apart as often as not, and all blocks at one k ask the same few channels (linear_rows.hip has figures). The last two
  // pieces stay the last.
  const unsigned count = last > first ? last - first : 0, plain = count > 2 ? count - 2 : 0;
  const unsigned begin = args.rotate && plain > 0 ? at.bx % plain : 0;
  x_next += (size_t)begin * x_step;
  y_next += (size_t)begin * y_step;
  unsigned piece_next = first + begin, copied = 0;
  // Copy n of the wave's COPIES of the next piece. `end`: it may be one of the last two pieces of K.
  auto copy_one = [&](unsigned slot, auto copy, auto end) {
    constexpr int n = decltype(copy)::value;
    constexpr bool of_x = n < X_COPIES, contiguous = of_x ? X_ROWS : Y_ROWS;
    constexpr int q = of_x ? n : n - X_COPIES;
    const char *const from = of_x ? x_next : y_next;
    const unsigned to = uniform(lds_base + slot * SLOT_BYTES + (of_x ? 0 : X_BYTES) + (wave + q * WAVES) * 1024);
    if constexpr (!decltype(end)::value) {
      load_1k_to_lds(uniform(from), offset[n], to);
    } else {
      const char *lane_from = from + offset[n];
      const Tail tail = of_x ? args.x_tail : args.y_tail;
      if constexpr (contiguous) {
        const unsigned k = piece_next * kPiece + chunk * 8;
        if (k + 8 > k_all && k_all >= 8) lane_from -= (size_t)(k + 8 - k_all) * 2;
        if (tail.copy && lane_from + 16 > tail.end) lane_from = tail.copy + 32 - (tail.end - lane_from);
        if (k >= k_all) lane_from = zeros;
      } else {
        const unsigned pitch = of_x ? args.x_pitch : args.y_pitch;
        const unsigned row = (unsigned)((wave + q * WAVES) * 64 + lane) / (of_x ? BX / 8 : BY / 8);
        const unsigned k = piece_next * kPiece + row;
        bool inside = k < k_all;
        if constexpr (Y_ROWS) {      // (as Y's chunk at the end of its rows)
          const unsigned chunk_end = (k & ~7u) + 8;
          if (chunk_end > k_all && k_all >= 8) {
            inside = chunk_end - 8 < k_all;
            lane_from -= (size_t)(chunk_end - k_all) * pitch;
          }
        }
        if (tail.copy && lane_from + 16 > tail.end) lane_from = tail.copy + 32 - (tail.end - lane_from);
        if (!inside) lane_from = zeros;
      }
      load_1k_to_lds_by_lane(lane_from, to);
    }
  };
  auto advance = [&]() {
    x_next += x_step;
    y_next += y_step;
    ++piece_next;
    ++copied;
    auto jump = [&](int pieces) {
      x_next += (long long)pieces * (long long)x_step;
      y_next += (long long)pieces * (long long)y_step;
      piece_next += pieces;
    };
    if (copied == plain - begin) jump(-(int)plain);
    if (copied == plain) jump((int)(plain - begin));
  };
  const std::true_type may_end{};

  // ---- fragments ----
  const int fr = lane & 15, g = lane >> 4;
  const unsigned frag0 = fr * 128 + ((g ^ (fr & 7)) << 4), frag1 = fr * 128 + (((g + 4) ^ (fr & 7)) << 4);
  const unsigned k_row = 8 * g + (fr >> 2);
  const unsigned x_lane = k_row * (BX * 2) + (fr & 3) * (8 * NT), x_swizzle = unit_swizzle<BX * 2, UNIT_X>(k_row) * UNIT_X;
  const unsigned y_lane = k_row * (BY * 2) + (fr & 3) * 8, y_swizzle = unit_swizzle<BY * 2, 32>(k_row) * 32;
  (void)frag0, (void)frag1, (void)x_lane, (void)x_swizzle, (void)y_lane, (void)y_swizzle;
  auto read_along = [&](const char *p) {
    const int4_t a = *reinterpret_cast<const int4_t *>(p + frag0), b = *reinterpret_cast<const int4_t *>(p + frag1);
    return Fragment(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto read_across = [&](unsigned address, auto row_bytes) {
    constexpr int ROW = decltype(row_bytes)::value;
    typedef int int2_t __attribute__((ext_vector_type(2)));
    Fragment f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const auto from = (__attribute__((address_space(3))) short4_t *)(uintptr_t)(address + (q * 32 + h * 4) * ROW);
        const int2_t v = __builtin_bit_cast(int2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(from));
        f[q * 4 + h * 2] = v[0];
        f[q * 4 + h * 2 + 1] = v[1];
      }
    }
    return f;
  };
  auto read_x = [&](unsigned slot, int i) {
    if constexpr (X_ROWS) {
      return read_along(lds + slot * SLOT_BYTES + (wx * TX + i * 16) * 128);
    } else {
      const unsigned unit = (unsigned)(wx * TX + i / NT * NT * 16) * 2;     // bytes
      return read_across(lds_base + slot * SLOT_BYTES + x_lane + (unit ^ x_swizzle) + i % NT * 8, std::integral_constant<int, BX * 2>{});
    }
  };
  auto read_y = [&](unsigned slot, int j) {
    if constexpr (Y_ROWS) {
      return read_along(lds + slot * SLOT_BYTES + X_BYTES + (wy * TY + j * 16) * 128);
    } else {
      const unsigned unit = (unsigned)(wy * TY + j * 16) * 2;
      return read_across(lds_base + slot * SLOT_BYTES + X_BYTES + y_lane + (unit ^ y_swizzle), std::integral_constant<int, BY * 2>{});
    }
  };

  float4_t acc[NY][NX];
#pragma unroll
  for (int j = 0; j < NY; ++j) {
#pragma unroll
    for (int i = 0; i < NX; ++i) acc[j][i] = 0.f;
  }

  // ---- K loop ----
  // A step is the products of one X tile with JJ Y tiles. What a step needs is read while the ones before it run: the
  // fragment of X tile i + 1 behind the first products of tile i; the fragments of Y and the first X fragment of the
  // next piece behind the products of the last tile, at whose start the wave waits for its copies of that piece and passes the
  // barrier. Behind it nobody reads this piece's slot any more: the copies of the piece that is to lie there go out at once, BEHIND of
  // them behind the last tile's products, the others behind the next piece's first ones, so that they have a whole piece's time
  // (8192^3 with all of them in the next piece: 845 us). The order is written out, as in real_gemm.h.
  constexpr int JJ = NY % 2 ? 1 : 2, SPT = NY / JJ, STEPS = NX * SPT;
  constexpr int COPY_STEPS = STEPS - SPT, PER_STEP = 1;
  constexpr int BEHIND = COPY_STEPS == 0 || SPT * PER_STEP > COPIES ? COPIES : SPT * PER_STEP;
  constexpr int PER_BEHIND = (BEHIND + SPT - 1) / SPT, REST = COPIES - BEHIND;
  constexpr int PER_REST = REST == 0 ? 0 : REST <= COPY_STEPS * PER_STEP ? PER_STEP : (REST + COPY_STEPS - 1) / (COPY_STEPS ? COPY_STEPS : 1);
  const unsigned n = count;
  if (n > 0) {
#pragma unroll
    for (int t = 0; t < SLOTS - 1; ++t) {
      if ((unsigned)t < n) {
        static_for<COPIES>([&](auto c) { copy_one(t, c, may_end); });
        advance();
      }
    }
    Fragment y[NY], x[2];
    if (n >= (unsigned)SLOTS) {   // (what piece -1 would have begun)
      static_for<BEHIND>([&](auto c) { copy_one(SLOTS - 1, c, may_end); });
      real::wait_copies_then_barrier<COPIES *(SLOTS - 2) + BEHIND>();
    } else {
      real::wait_copies_then_barrier<0>();
    }
    unsigned slot = 0, before = SLOTS - 1;      // of this piece, of the one before
    x[0] = read_x(0, 0);
#pragma unroll
    for (int j = 0; j < NY; ++j) y[j] = read_y(0, j);
    // Piece t. What is copied: kAll the rest of piece t + SLOTS - 1 and the first of piece t + SLOTS; kEnds the same, where these may
    // be the last ones of K; kRest the rest only; kNothing; kLast nothing, and no piece follows.
    enum { kAll, kEnds, kRest, kNothing, kLast };
    auto piece = [&](auto what) {
      constexpr int WHAT = decltype(what)::value;
      constexpr bool LAST = WHAT == kLast, COPY_REST = WHAT <= kRest, COPY_BEHIND = WHAT <= kEnds;
      const unsigned next = slot + 1 == SLOTS ? 0 : slot + 1;
      const std::integral_constant<bool, WHAT != kAll> end{};
      // Values of the last chunk along k that have been multiplied already, or lie beyond a row of less than 8
      Fragment keep;
      auto clear = [&](Fragment &f) {
        if constexpr (LAST && KIND != kWeights) f &= keep;
      };
      if constexpr (LAST && KIND != kWeights) {
        const unsigned left = k_all - (last - 1) * kPiece, ends = left < kPiece ? left % 8 : 0;
        const unsigned from = k_all >= 8 ? (8 - ends) % 8 : 0, until = k_all >= 8 ? 8 : ends;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const unsigned e = d % 4 * 2;
          const int mask = (e >= from && e < until ? 0xffff : 0) | (e + 1 >= from && e + 1 < until ? (int)0xffff0000 : 0);
          keep[d] = ends && (unsigned)(g + d / 4 * 4) == left / 8 ? mask : -1;
        }
#pragma unroll
        for (int j = 0; j < NY; ++j) clear(y[j]);
        clear(x[0]);
      }
      static_for<STEPS>([&](auto step) {
        constexpr int m = step, i = m / SPT, js = m % SPT, to = (i + 1) % 2;
        constexpr bool at_end = i == NX - 1;
        CCGLIB_PIN;
        if constexpr (at_end && js == 0) {
          if constexpr (COPY_REST) advance();
          // (as many later pieces are on their way; behind the last copies all of them have to have arrived)
          if constexpr (!LAST) real::wait_copies_then_barrier<COPY_REST ? COPIES *(SLOTS - 2) : 0>();
        }
        if constexpr (js == 0) {
          if constexpr (!at_end) {
            x[to] = read_x(slot, i + 1);
          } else if constexpr (!LAST) {
            x[to] = read_x(next, 0);
          }
        }
#pragma unroll
        for (int h = 0; h < JJ; ++h) pin(y[js * JJ + h]);
        auto products = [&](int q) {
#pragma unroll
          for (int h = 0; h < JJ; ++h) {
            const int j = js * JJ + h;
            acc[j][i] = mfma<TYPE>(x[i % 2], y[j], acc[j][i], q);
          }
#pragma unroll
          for (int h = 0; h < JJ; ++h) pin(acc[js * JJ + h][i]);
          CCGLIB_PIN;
        };
        products(0);
        if constexpr (!at_end && COPY_REST) {
          constexpr int c0 = m * PER_REST < REST ? m * PER_REST : REST, c1 = (m + 1) * PER_REST < REST ? (m + 1) * PER_REST : REST;
          static_for<c1 - c0>([&](auto c) { copy_one(before, std::integral_constant<int, BEHIND + c0 + decltype(c)::value>{}, end); });
        }
        if constexpr (at_end && COPY_BEHIND) {
          constexpr int c0 = js * PER_BEHIND < BEHIND ? js * PER_BEHIND : BEHIND;
          constexpr int c1 = (js + 1) * PER_BEHIND < BEHIND ? (js + 1) * PER_BEHIND : BEHIND;
          static_for<c1 - c0>([&](auto c) { copy_one(slot, std::integral_constant<int, c0 + decltype(c)::value>{}, end); });
        }
        CCGLIB_PIN;
        products(1);
        if constexpr (at_end && !LAST) {
#pragma unroll
          for (int h = 0; h < JJ; ++h) y[js * JJ + h] = read_y(next, js * JJ + h);
        }
        if constexpr (js == SPT - 1 && !at_end) clear(x[to]);
      });
      if constexpr (NX % 2 == 1) x[0] = x[1];   // (the next piece's first tile, where its predecessor was in use)
      before = slot;
      slot = next;
    };
    // (pieces of K's end, or of an operand's, are among the last two)
    unsigned t = 0;
#pragma unroll 1
    for (; t + SLOTS < plain; ++t) piece(std::integral_constant<int, kAll>{});
#pragma unroll 1
    for (; t + SLOTS < n; ++t) piece(std::integral_constant<int, kEnds>{});
    if (t + SLOTS == n) {
      piece(std::integral_constant<int, kRest>{});
      ++t;
    }
#pragma unroll 1
    for (; t + 1 < n; ++t) piece(std::integral_constant<int, kNothing>{});
    piece(std::integral_constant<int, kLast>{});
  }

  // ---- parts of K joined: in the order of the parts, whichever block arrives last (as in real_gemm.h) ----
  if (args.parts > 1) {
    typedef unsigned long long piece_t;
    constexpr int PIECES = 2;     // of a lane's four sums
    constexpr size_t BLOCK = (size_t)BX * BY / PIECES;
    piece_t *const all = reinterpret_cast<piece_t *>(args.partial) + (size_t)at.tile * args.parts * BLOCK;
    piece_t *const mine = all + at.part * BLOCK + threadIdx.x;
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
          const float pair[2] = {acc[j][i][2 * h], acc[j][i][2 * h + 1]};
          __hip_atomic_store(mine + ((j * NX + i) * PIECES + h) * (64 * WAVES), __builtin_bit_cast(piece_t, pair), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the stores have arrived
    __syncthreads();
    unsigned *const flag = reinterpret_cast<unsigned *>(lds);
    if (threadIdx.x == 0) {
      const unsigned before = __hip_atomic_fetch_add(args.arrived + at.tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *flag = before + 1 == args.parts;
      if (before + 1 == args.parts) {
        __hip_atomic_store(args.arrived + at.tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    __syncthreads();
    if (*flag == 0) return;
    const piece_t *from = all + threadIdx.x;
#pragma unroll 1
    for (unsigned p = 0; p < args.parts; ++p, from += BLOCK) {
#pragma unroll
      for (int j = 0; j < NY; ++j) {
#pragma unroll
        for (int i = 0; i < NX; ++i) {
#pragma unroll
          for (int h = 0; h < PIECES; ++h) {
            const piece_t u = __hip_atomic_load(from + ((j * NX + i) * PIECES + h) * (64 * WAVES), __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT);
            const float lo = __builtin_bit_cast(float, (unsigned)u), hi = __builtin_bit_cast(float, (unsigned)(u >> 32));
            acc[j][i][2 * h] = p == 0 ? lo : acc[j][i][2 * h] + lo;
            acc[j][i][2 * h + 1] = p == 0 ? hi : acc[j][i][2 * h + 1] + hi;
          }
        }
        CCGLIB_PIN;      // (all loads at once would take more registers than there are)
      }
    }
  }

  // ---- epilogue ----
  constexpr int N = 4 * NT;
#pragma unroll
  for (int i = 0; i < NX; i += NT) {
    if constexpr (KIND == kWeights && NT == 2 && TX != 64) {
      const unsigned x = x0 + wx * TX + i * 16;
      if (params.wide && x + 32 <= args.nx) {
        CCGLIB_PIN;
#pragma unroll
        for (int j = 0; j < NY; ++j) {
          const unsigned row = y0 + wy * TY + j * 16 + fr;
          if (row < ny) store_wide<TX % 64 == 0>(params, at.group, row, x + g * 4, acc[j][i], acc[j][i + 1]);
        }
        continue;
      }
    }
    const unsigned x = x0 + wx * TX + i * 16 + g * N, left = x < args.nx ? args.nx - x : 0;
    CCGLIB_PIN;      // (one tile's loads at a time: all of them at once take more registers than there are)
    if (left == 0) continue;
    float bias[N] = {};
    if (KIND == kOutput && params.bias) {
      load_row(reinterpret_cast<const typename Value<TYPE>::type *>(params.bias) + (size_t)at.group * args.nx + x, left, bias);
    }
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      const unsigned row = y0 + wy * TY + j * 16 + fr;
      if (row >= ny) continue;
      float v[N];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * t + e] = acc[j][i + t][e];
      }
      store_sums<TYPE, KIND, TX % 64 == 0>(params, bias, at.group, Y_ROWS ? at.rows.first + row : row, x, left, v);
    }
  }
}

// Block `id` of `blocks` of a product.
template <int TYPE, int KIND, int BX, int BY, int WX, int WY, int SLOTS>
__device__ __forceinline__ void product(const Args &args, const StoreParams &params, char *lds, unsigned id, unsigned blocks) {
  const Place at = place<KIND, BY, false>(args, id, blocks);
  if (!at.none) product_at<TYPE, KIND, BX, BY, WX, WY, SLOTS>(args, params, lds, at, at.bx * BX, at.by * BY);
}

template <int TYPE, int KIND, int BX, int BY, int WX, int WY, int SLOTS, int WAVES_PER_EU>
__global__ __launch_bounds__(64 * WX * WY, WAVES_PER_EU) void gemm_linear(Args args, StoreParams params) {
  __shared__ __attribute__((aligned(256))) char lds[kLdsBytes<BX, BY, SLOTS>];
  product<TYPE, KIND, BX, BY, WX, WY, SLOTS>(args, params, lds, blockIdx.x, gridDim.x);
}

// 256 x 256 blocks whose last round, if it leaves half of the units idle, is one of 128 x 256 or 128 x 128 pieces. K is not cut, and rows
// of groups are not its length.
template <int TYPE, int KIND> __global__ __launch_bounds__(512, 2) void gemm_linear_cut(Args args, StoreParams params) {
  __shared__ __attribute__((aligned(256))) char lds[kLdsBytes<128, 256, 3>];
  static_assert(kLdsBytes<256, 256, 2> <= sizeof lds && kLdsBytes<128, 128, 4> <= sizeof lds, "one after the other");
  const Place at = place<KIND, 256, true>(args, blockIdx.x, gridDim.x);
  if (at.none) return;
  unsigned x0 = at.bx * 256, y0 = at.by * 256;
  if (at.cut == 1) {
    product_at<TYPE, KIND, 256, 256, 2, 4, 2>(args, params, lds, at, x0, y0);
    return;
  }
  x0 += at.piece % 2 * 128;
  y0 += at.piece / 2 * 128;
  if (x0 >= args.nx || y0 >= (KIND != kWeights && args.offsets ? at.rows.count : args.ny)) return;
  if (at.cut == 2) {
    product_at<TYPE, KIND, 128, 256, 2, 4, 3>(args, params, lds, at, x0, y0);
  } else {
    product_at<TYPE, KIND, 128, 128, 4, 2, 4>(args, params, lds, at, x0, y0);
  }
}

// Block shapes: BX x BY, waves, ring, waves a SIMD. (128 x 128 with four waves, two blocks to a unit, was nowhere the fastest of 34 problems
// in three products each; without any other of these the best choice is 0.6 to 2.7 % behind in the mean.)
#define CCGLIB_LINEAR_SHAPES(DO) \
  DO(0, 256, 256, 2, 4, 2, 2)    \
  DO(1, 64, 64, 2, 2, 4, 2)      \
  DO(2, 64, 32, 4, 1, 6, 2)      \
  DO(3, 128, 128, 4, 2, 4, 2)    \
  DO(4, 192, 192, 4, 2, 3, 2)    \
  DO(5, 128, 256, 2, 4, 3, 2)
constexpr int kCutShape = 6;   // gemm_linear_cut

template <int TYPE, int KIND> hipError_t launch_gemm(int shape, unsigned grid, const Args &a, const StoreParams &s, hipStream_t stream);
#define CCGLIB_DECLARE(TYPE, KIND) \
  template <> hipError_t launch_gemm<TYPE, KIND>(int shape, unsigned grid, const Args &a, const StoreParams &s, hipStream_t stream);
CCGLIB_DECLARE(kFloat16, kOutput)
CCGLIB_DECLARE(kFloat16, kInput)
CCGLIB_DECLARE(kFloat16, kWeights)
CCGLIB_DECLARE(kBfloat16, kOutput)
CCGLIB_DECLARE(kBfloat16, kInput)
CCGLIB_DECLARE(kBfloat16, kWeights)
#undef CCGLIB_DECLARE

// y of few rows (linear_rows.hip): blocks of 16 columns and kRowsOfX rows
constexpr int kRowsOfX = 16;
size_t linear_rows_blocks(size_t n);
hipError_t launch_linear_rows(int type, unsigned grid, const Args &a, const StoreParams &s, hipStream_t stream);

#ifdef CCGLIB_LINEAR_KIND
template <>
hipError_t launch_gemm<CCGLIB_LINEAR_TYPE, CCGLIB_LINEAR_KIND>(int shape, unsigned grid, const Args &a, const StoreParams &s,
                                                               hipStream_t stream) {
  switch (shape) {
#define CCGLIB_CASE(ID, BX, BY, WX, WY, SLOTS, EU)                                                                               \
  case ID:                                                                                                                       \
    gemm_linear<CCGLIB_LINEAR_TYPE, CCGLIB_LINEAR_KIND, BX, BY, WX, WY, SLOTS, EU><<<grid, 64 * WX * WY, 0, stream>>>(a, s); \
    break;
    CCGLIB_LINEAR_SHAPES(CCGLIB_CASE)
#undef CCGLIB_CASE
  case kCutShape:
    gemm_linear_cut<CCGLIB_LINEAR_TYPE, CCGLIB_LINEAR_KIND><<<grid, 512, 0, stream>>>(a, s);
    break;
  }
  return hipGetLastError();
}
#endif

}  // namespace linear
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_LINEAR_GEMM_H_
