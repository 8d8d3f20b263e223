// Products of real matrices whose rows are both contiguous along the summed index:
//   D[y][x] = sum_k X[x][k] Y[y][k],   x the contiguous axis of D,
// on the matrix cores, for the operators that need more than a plain product: 8-bit operands with scales
// (scaled_gemm.hip) and the symmetric chains of Newton-Schulz steps (orthogonalize.hip).
//
// Rows are walked in pieces of 128 bytes: 128 values of 8 bits, which is the length that one scale covers
// and what one 16x16x128 instruction multiplies, or 64 values of 16 bits, two 16x16x32 instructions. Every piece of a
// row is a whole cache line, and the two kinds share the loader, the LDS layout and the fragment reads: a lane
// reads the 16-byte chunks g and g + 4 (g = lane / 16) of row lane % 16. For 8 bits that permutes K inside the piece,
// in the same way for both operands.
//
// LDS: a ring of SLOTS pieces. The copies go straight to LDS (global_load_lds_dwordx4, 8 rows of 128 bytes each),
// chunk c of row r at position c ^ (r & 7), which keeps the fragment reads free of bank conflicts. One barrier a
// piece: a wave waits for its own copies, passes the barrier, and refills the slot that everybody has left.
//
// Sums: X supplies the instruction's rows, Y its columns, and the rows of X are permuted inside groups of 16 NT
// (by the copies), so that a lane's registers hold 4 NT consecutive x at one y: wide stores.
//
// What bounds it: in large products the matrix instructions are busy 40 to 60 % of the cycles, at a clock that the power limit
// has down to 2.0 to 2.2 GHz of 2.4, next to LDS reads, copies, barriers and, with float scales, the vector additions. 8192^3: float
// scales for 128 x 128 458 us, 2400 TFLOP/s; for rows 541, 2030; e8m0 440, 2500 (a library product of the same values without block
// scales 329, 3340); 8 bits as fp16 901 to 1031, 1070 to 1220; fp16 P X of 4096 x 8192 219, 1250 (library 1570). Other cards
// are up to 6 % slower in all of them. A single row: 8192 x 8192 bytes in 14 us out of the last-level cache, in 19.5 (3.4 TB/s) where
// they come from memory. Blocks that are alone on a unit: one round trip a piece, which is what the deeper rings are for.
#ifndef CCGLIB_AMD_REAL_GEMM_H_
#define CCGLIB_AMD_REAL_GEMM_H_

#include <type_traits>
#include <utility>

#include "gemm_device.h"

namespace ccglib_amd {
namespace real {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef int int8x_t __attribute__((ext_vector_type(8)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// How operands are multiplied.
enum Mode {
  kScaledBlocks = 0,  // 8 bits, float scales; X has one scale for 128 rows
  kScaledRows = 1,    // 8 bits, float scales; X has one for each row (or is given so)
  kScaledE8m0 = 2,    // 8 bits, power-of-two scales, applied by the matrix instruction
  // The same, the 8-bit values turned into fp16 (which holds every one of them) in registers and multiplied by the
  // fp16 instruction. The 8-bit one aligns the products of eight neighbours in K to the largest of them and drops
  // what lies below 2^-13 of that: 1.5e-5 of a sum of 128 products of N(0, 1) values, 3e-5 to 9e-5 where some columns are
  // much larger than others. That is far below the rounding to 16 bits (2e-4 and 1.7e-3), but not below that to 32.
  kWideBlocks = 3,
  kWideRows = 4,
  kWideE8m0 = 5,
  kHalf = 6,          // fp16
  kHalfPairs = 7      // every value as the sum of two fp16, the second one times 2^11
};

constexpr int kPieceBytes = 128;

struct Args {
  const char *x, *y;             // rows of bytes
  unsigned nx, ny, batch;
  unsigned x_pitch, y_pitch;     // bytes from row to row
  size_t x_batch, y_batch;       // bytes from matrix to matrix
  size_t x_plane, y_plane;       // kHalfPairs: bytes from the first parts to the second ones
  unsigned k_bytes;              // bytes of a row that are read, a multiple of 16
  unsigned pieces;               // ceil(k_bytes / 128)
  unsigned blocks_x, blocks_y;
  unsigned symmetric;            // D is: blocks with block_x <= block_y only (BX = BY)
  // scales [batch][pieces][pitch], of 4 bytes or 1; row r has number r >> shift
  const char *x_scales, *y_scales;
  unsigned x_scale_pitch, y_scale_pitch, x_shift, y_shift;
  // K in `parts` pieces of pieces_per_part, each a block of its own: sums of all but the last block that arrives go
  // through `partial`
  unsigned parts, pieces_per_part;
  float *partial;
  unsigned *arrived;             // per block of D, zero between launches
};

// 16 bytes of zeros that lanes beyond the end of a row read
static __device__ __attribute__((aligned(16))) char g_zeros[16];

template <int MODE> struct ModeTraits {
  static constexpr bool kScaled = MODE <= kWideE8m0;
  static constexpr bool kWide = MODE >= kWideBlocks && MODE <= kWideE8m0;
  static constexpr bool kBlocks = MODE == kScaledBlocks || MODE == kWideBlocks;
  static constexpr int kPlanes = MODE == kHalfPairs ? 2 : 1;
  static constexpr int kSums = MODE == kHalfPairs ? 2 : 1;
  static constexpr int kScaleBytes = MODE == kScaledE8m0 || MODE == kWideE8m0 ? 1 : 4;
};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 scales to LDS, a dword each (those of one byte zero-extended)
template <int BYTES>
__device__ __forceinline__ void load_scales_to_lds(const char *base, unsigned lane_offset, unsigned lds_address) {
  unsigned long long base_here;
  if constexpr (BYTES == 4) {
    asm volatile(
        "s_mov_b64 %0, %3\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, %0"
        : "=&s"(base_here) : "s"(lds_address), "v"(lane_offset), "s"(base) : "memory", "m0");
  } else {
    asm volatile(
        "s_mov_b64 %0, %3\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %2, %0"
        : "=&s"(base_here) : "s"(lds_address), "v"(lane_offset), "s"(base) : "memory", "m0");
  }
}
#pragma clang diagnostic pop

template <int N> __device__ __forceinline__ void wait_copies_then_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// 32 bytes of a row: two 16-byte chunks
typedef int8x_t Fragment;
__device__ __forceinline__ half8_t half_of(const Fragment &f, int q) {
  const int4_t v = q == 0 ? __builtin_shufflevector(f, f, 0, 1, 2, 3) : __builtin_shufflevector(f, f, 4, 5, 6, 7);
  return __builtin_bit_cast(half8_t, v);
}

// FX, FY: format codes of 8-bit operands (0 e4m3, 1 e5m2)
template <int FX, int FY>
__device__ __forceinline__ float4_t mfma8(const Fragment &x, const Fragment &y, float4_t c, int sx, int sy) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, FX, FY, 0, sx, 0, sy);
}

// A lane's 32 values of 8 bits as fp16, four operands of the fp16 instruction
struct WideFragment {
  half8_t v[4];
};
// (word w, of eight: four values)
template <int FORMAT> __device__ __forceinline__ void widen_word(const Fragment &f, WideFragment &to, int w) {
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  const unsigned word = (unsigned)f[w];
  half2_t lo, hi;
  if constexpr (FORMAT == 0) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, true);
  } else {   // (e5m2 is the upper half of fp16)
    lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(word, word, 0x010c000cu));
    hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(word, word, 0x030c020cu));
  }
  const int q = w / 2, at = w % 2 * 4;
  to.v[q][at] = lo[0];
  to.v[q][at + 1] = lo[1];
  to.v[q][at + 2] = hi[0];
  to.v[q][at + 3] = hi[1];
}
template <int FORMAT> __device__ __forceinline__ WideFragment widened(const Fragment &f) {
  WideFragment r;
#pragma unroll
  for (int w = 0; w < 8; ++w) widen_word<FORMAT>(f, r, w);
  return r;
}
// 2^(byte - 127); NaN for 255, which stands for no number
__device__ __forceinline__ float power_of_two(unsigned byte) {
  return byte == 255 ? __builtin_nanf("") : __builtin_ldexpf(0x1p-127f, (int)byte);
}

__device__ __forceinline__ float4_t mfma16(const Fragment &x, const Fragment &y, float4_t c, int q) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(half_of(x, q), half_of(y, q), c, 0, 0, 0);
}

// Nothing moves across: neither instructions, when they are put in order, nor reads of LDS, when they are selected
#define CCGLIB_PIN                      \
  do {                                  \
    asm volatile("" ::: "memory");      \
    __builtin_amdgcn_sched_barrier(0);  \
  } while (0)
// What computes the value comes before this place, what uses it comes behind it (arithmetic has no other order than that of
// its operands until the instructions have been selected)
template <typename T> __device__ __forceinline__ void pin(T &value) { asm volatile("" : "+v"(value)); }
__device__ __forceinline__ void pin(WideFragment &value) {
#pragma unroll
  for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(value.v[q]));
}

__device__ __forceinline__ void pin_scalar(const char *&p) { asm volatile("" : "+s"(p)); }

template <int N, typename F, int... I> __device__ __forceinline__ void static_for(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void static_for(F &&f) {
  static_for<N>(f, std::make_integer_sequence<int, N>{});
}

// (the same in every lane: say so where it goes to a scalar register of an asm statement)
__device__ __forceinline__ const char *uniform(const char *p) {
  const unsigned long long u = (unsigned long long)p;
  const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)u);
  const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32));
  return (const char *)(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ unsigned uniform(unsigned u) { return (unsigned)__builtin_amdgcn_readfirstlane((int)u); }

// Which block of D, and which piece of K, a workgroup has.
struct Place {
  unsigned b, bx, by, part, tile;
};
__device__ __forceinline__ Place place(const Args &a) {
  const unsigned per_matrix = a.symmetric ? a.blocks_y * (a.blocks_y + 1) / 2 : a.blocks_x * a.blocks_y;
  const unsigned id = xcd_remap(blockIdx.x, gridDim.x);
  Place p;
  const unsigned t = id % per_matrix, rest = id / per_matrix;
  p.part = rest % a.parts;
  p.b = rest / a.parts;
  p.tile = p.b * per_matrix + t;
  if (a.symmetric) {
    unsigned y = (unsigned)((__builtin_sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (y * (y + 1) / 2 > t) --y;
    while ((y + 1) * (y + 2) / 2 <= t) ++y;
    p.by = y;
    p.bx = t - y * (y + 1) / 2;
  } else {
    // groups of four block rows, y fastest: the blocks that an XCD works on at one time share rows of X and of Y
    constexpr unsigned GROUP = 4;
    const unsigned g = t / (GROUP * a.blocks_x), in = t - g * GROUP * a.blocks_x;
    const unsigned rows = a.blocks_y - g * GROUP < GROUP ? a.blocks_y - g * GROUP : GROUP;
    p.by = g * GROUP + in % rows;
    p.bx = in / rows;
  }
  p.b = (unsigned)__builtin_amdgcn_readfirstlane((int)p.b);
  p.bx = (unsigned)__builtin_amdgcn_readfirstlane((int)p.bx);
  p.by = (unsigned)__builtin_amdgcn_readfirstlane((int)p.by);
  p.part = (unsigned)__builtin_amdgcn_readfirstlane((int)p.part);
  p.tile = (unsigned)__builtin_amdgcn_readfirstlane((int)p.tile);
  return p;
}

template <int MODE, int BX, int BY, int WX, int WY, int SLOTS> struct Shape {
  static constexpr int kWaves = WX * WY;
  static constexpr int kPlanes = ModeTraits<MODE>::kPlanes;
  static constexpr int kXBytes = BX * kPieceBytes * kPlanes, kYBytes = BY * kPieceBytes * kPlanes;
  static constexpr int kScaleBytes = ModeTraits<MODE>::kScaled ? (BX + BY + 63) / 64 * 64 * 4 : 0;
  static constexpr int kSlotBytes = kXBytes + kYBytes + kScaleBytes;
  static constexpr int kLdsBytes = SLOTS * kSlotBytes;
};

// N neighbouring values of type T from `to` on, of which `left` are inside the row; `to` is aligned to its element only.
template <typename T, int N> __device__ __forceinline__ void store_row(T *to, unsigned left, const float (&v)[N]) {
  constexpr int E = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
  typedef T piece_t __attribute__((ext_vector_type(E)));
  typedef piece_t piece_unaligned_t __attribute__((aligned(sizeof(T))));
  if (left >= (unsigned)N) {
#pragma unroll
    for (int i = 0; i < N; i += E) {
      piece_t w;
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = (T)v[i + e];
      *reinterpret_cast<piece_unaligned_t *>(to + i) = w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if ((unsigned)e < left) to[e] = (T)v[e];
    }
  }
}

// What an epilogue is given: 16 NT columns of a wave's tile, from x on, of rows y + 16 j + lane % 16; a lane's values are
// N = 4 NT neighbours from x + N (lane / 16) on. `lds`: kGroupLds bytes for this wave alone.
struct Group {
  unsigned b, y, x;
  int lane;
  bool mirror;      // D is symmetric, and this block's transpose has no block of its own
  char *lds;
};
// Rows of a wave's group in LDS, transposed, of 16-bit values: 16 bytes apart from a multiple of 128 bytes, which spreads the
// pieces of a column over the banks
template <int NY> constexpr int kGroupPitch = NY * 16 * 2 + 16;

// Epilogue: has `Params`, a constructor from them, and
//   template <int NY, int N> void store(const Group &, float (&v)[NY][N])
template <int MODE, int FX, int FY, int BX, int BY, int WX, int WY, int SLOTS, int WAVES_PER_EU, class Epilogue>
__global__ __launch_bounds__(64 * WX * WY, WAVES_PER_EU) void gemm_real(Args args, typename Epilogue::Params params) {
  using S = Shape<MODE, BX, BY, WX, WY, SLOTS>;
  using T = ModeTraits<MODE>;
  constexpr int WAVES = WX * WY, PLANES = T::kPlanes;
  constexpr int TX = BX / WX, TY = BY / WY, NX = TX / 16, NY = TY / 16;
  // (a lane's neighbours in D: 16 bytes of 16 or 32 bits each, so that a store instruction writes 64 bytes of a row at once)
  constexpr int NT = T::kWide || NX % 2 ? 1 : 2, GROUP_ROWS = 16 * NT;
  constexpr int X_COPIES = BX / 8 * PLANES, COPIES_ALL = X_COPIES + BY / 8 * PLANES;
  constexpr int OPERAND_COPIES = COPIES_ALL / WAVES;
  constexpr int SCALE_COPIES = T::kScaled ? (BX + BY + 63) / 64 : 0;
  constexpr int COPIES = OPERAND_COPIES + (T::kScaled ? 1 : 0);
  static_assert(BX / 8 % WAVES == 0 && BY / 8 % WAVES == 0 && SCALE_COPIES <= WAVES && NX % NT == 0, "shape");
  __shared__ __attribute__((aligned(256))) char lds[S::kLdsBytes];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wx = wave % WX, wy = wave / WX;
  const Place at = place(args);
  const unsigned x0 = at.bx * BX, y0 = at.by * BY;
  const unsigned first = at.part * args.pieces_per_part;
  const unsigned last = first + args.pieces_per_part < args.pieces ? first + args.pieces_per_part : args.pieces;
  const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

  // ---- copies ----
  const char *const x_base = args.x + (size_t)at.b * args.x_batch + (size_t)x0 * args.x_pitch;
  const char *const y_base = args.y + (size_t)at.b * args.y_batch + (size_t)y0 * args.y_pitch;
  const unsigned chunk = (unsigned)((lane & 7) ^ (lane >> 3));
  unsigned offset[OPERAND_COPIES];
#pragma unroll
  for (int n = 0; n < OPERAND_COPIES; ++n) {
    // (a wave's n-th copy of a piece: of which operand is known beforehand)
    const bool of_x = n < X_COPIES / WAVES;
    const int q = wave + (of_x ? n : n - X_COPIES / WAVES) * WAVES;
    const int row = (q % ((of_x ? BX : BY) / 8)) * 8 + (lane >> 3);
    unsigned want = row;
    if (of_x) {   // row `row` of LDS holds this row of the block
      const int in = row % GROUP_ROWS, t = in / 16, r = in % 16;
      want = row - in + (r >> 2) * (4 * NT) + t * 4 + (r & 3);
    }
    const unsigned most = (of_x ? args.nx - x0 : args.ny - y0) - 1;   // (rows past the end: never stored)
    offset[n] = (want < most ? want : most) * (of_x ? args.x_pitch : args.y_pitch) + chunk * 16;
  }
  unsigned scale_offset = 0;
  const char *scale_base = nullptr;
  unsigned scale_step = 0, scale_lds = 0;
  if constexpr (T::kScaled) {
    // 64 rows' scales a wave: first those of X, then those of Y (BX + BY may end inside the last 64)
    const unsigned j = (unsigned)wave % SCALE_COPIES, row = j * 64 + lane;
    const bool of_x = BX % 64 == 0 ? j * 64 < (unsigned)BX : row < (unsigned)BX;
    unsigned r = of_x ? x0 + row : y0 + row - BX;
    const unsigned most = (of_x ? args.nx : args.ny) - 1;
    r = (r < most ? r : most) >> (of_x ? args.x_shift : args.y_shift);
    scale_offset = r * T::kScaleBytes;
    scale_step = (of_x ? args.x_scale_pitch : args.y_scale_pitch) * T::kScaleBytes;
    scale_base = (of_x ? args.x_scales : args.y_scales) + (size_t)at.b * args.pieces * scale_step;
    scale_lds = j * 256;
  }
  // (kept in registers: its address is a scalar load, behind which the LDS reads would be waited for all together)
  const char *zeros = g_zeros;
  pin_scalar(zeros);
  // Where the next piece to be copied is, and the slot of LDS that it goes to
  const char *x_next = x_base + (size_t)first * kPieceBytes, *y_next = y_base + (size_t)first * kPieceBytes;
  const char *scales_next = scale_base + (size_t)first * scale_step;
  unsigned piece_next = first;
  // Copy n of the wave's COPIES of that piece. `end`: the piece may end inside its 128 bytes; what lies beyond is zero
  // (the copies of a piece have no branch, and of the two kinds of loop below only the last one asks).
  auto copy_one = [&](unsigned slot, auto copy, auto end) {
    constexpr int n = decltype(copy)::value;
    const unsigned to = lds_base + slot * S::kSlotBytes;
    if constexpr (T::kScaled && n == OPERAND_COPIES) {
      load_scales_to_lds<T::kScaleBytes>(uniform(scales_next), scale_offset, uniform(to + S::kXBytes + S::kYBytes + scale_lds));
    } else {
      constexpr bool of_x = n < X_COPIES / WAVES;
      constexpr int in = of_x ? n : n - X_COPIES / WAVES, plane = in / ((of_x ? BX : BY) / 8 / WAVES);
      const char *from = of_x ? x_next : y_next;
      if constexpr (plane > 0) from += of_x ? args.x_plane : args.y_plane;
      const unsigned at_lds = uniform(to + (wave + n * WAVES) * 1024);
      if constexpr (!decltype(end)::value) {
        load_1k_to_lds(uniform(from), offset[n], at_lds);
      } else {
        load_1k_to_lds_by_lane((size_t)piece_next * kPieceBytes + chunk * 16 < args.k_bytes ? from + offset[n] : zeros, at_lds);
      }
    }
  };
  auto advance = [&]() {
    x_next += kPieceBytes;
    y_next += kPieceBytes;
    if constexpr (T::kScaled) scales_next += scale_step;
    ++piece_next;
  };
  const std::true_type may_end{};
  static_assert(!T::kScaled || BX % 64 == 0, "scales of X fill whole copies");

  // ---- fragments ----
  const int fr = lane & 15, g = lane >> 4;
  const unsigned frag0 = fr * kPieceBytes + ((g ^ (fr & 7)) << 4), frag1 = fr * kPieceBytes + (((g + 4) ^ (fr & 7)) << 4);
  auto read = [&](unsigned slot, int from) {
    const char *p = lds + slot * S::kSlotBytes + from;
    const int4_t a = *reinterpret_cast<const int4_t *>(p + frag0), b = *reinterpret_cast<const int4_t *>(p + frag1);
    return Fragment(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  const int x_rows = wx * TX * kPieceBytes, y_rows = S::kXBytes + wy * TY * kPieceBytes;

  float4_t acc[T::kSums][NY][NX];
#pragma unroll
  for (int s = 0; s < T::kSums; ++s) {
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int i = 0; i < NX; ++i) acc[s][j][i] = 0.f;
    }
  }
  const float4_t zero = {0.f, 0.f, 0.f, 0.f};

  // ---- K loop ----
  // A step is the products of one X tile with JJ Y tiles. Everything that a step needs is read while the ones before it
  // run: the fragment of X tile i + 1 behind the first products of tile i; the fragments of Y, the scales and the first X
  // fragment of the next piece behind the products of the last tile, at whose start the wave waits for its copies of that
  // piece and passes the barrier. With float scales the sums of a step are added to C's LAG steps later. The order is
  // written out; left to itself the compiler reads, multiplies, waits and adds one tile after the other (8192^3: 587 us).
  constexpr bool FLOAT_SCALES = T::kScaled && MODE != kScaledE8m0;
  constexpr int JJ = MODE <= kScaledE8m0 ? 1 : 2;     // (two sums in turn where several instructions add to one)
  constexpr int SPT = NY / JJ, STEPS = NX * SPT;
  constexpr int LAG = T::kWide ? 1 : 2, RING = 2 * LAG;
  constexpr bool CARRY = STEPS % RING == 0;           // the last sums of a piece are added during the next one
  // Copies go out behind the products before the last tile's, a few at a time: all of them lie in front of the wait there,
  // which counts on it
  constexpr int COPY_STEPS = STEPS - SPT, PER_STEP = COPY_STEPS > 0 ? (COPIES + COPY_STEPS - 1) / COPY_STEPS : 0;
  static_assert(NY % JJ == 0 && (!FLOAT_SCALES || SPT >= LAG), "steps");
  const unsigned n = last > first ? last - first : 0;
  if (n > 0) {
#pragma unroll
    for (int t = 0; t < SLOTS - 1; ++t) {
      if ((unsigned)t < n) {
        static_for<COPIES>([&](auto c) { copy_one(t, c, may_end); });
        advance();
      }
    }
    using Operand = typename std::conditional<T::kWide, WideFragment, Fragment>::type;
    Operand y[PLANES][NY], x[2][PLANES];
    Fragment raw_x, raw_y[T::kWide ? NY : 1];   // (8 bits that become fp16)
    // (scales are read a while before they are needed, and turned into what is needed only then)
    float s[NY], s_old[RING * JJ];      // scales of Y (times X's where that is one number)
    float sy_read[NY], sx_read = 0.f;
    float4_t sx[2];                     // scales of a lane's rows of X tile i
    int e8[NY], e8x[2];                 // e8m0: bytes for the instruction
    float4_t part[RING][JJ];
    (void)s, (void)s_old, (void)sy_read, (void)sx_read, (void)e8, (void)e8x, (void)sx, (void)part, (void)raw_x, (void)raw_y;
    auto scale = [](float stored) {
      return T::kScaleBytes == 1 ? power_of_two(__builtin_bit_cast(unsigned, stored)) : stored;
    };
    auto scales_at = [&](unsigned slot) { return lds + slot * S::kSlotBytes + S::kXBytes + S::kYBytes; };
    auto read_scales_y = [&](unsigned slot) {
      if constexpr (T::kScaled) {
        const float *const sxp = reinterpret_cast<const float *>(scales_at(slot)) + wx * TX;
        const float *const syp = reinterpret_cast<const float *>(scales_at(slot)) + BX + wy * TY;
#pragma unroll
        for (int j = 0; j < NY; ++j) sy_read[j] = syp[j * 16 + fr];
        if constexpr (T::kBlocks) sx_read = sxp[0];
      }
    };
    auto take_scales_y = [&]() {
#pragma unroll
      for (int j = 0; j < NY; ++j) {
        if constexpr (FLOAT_SCALES) s[j] = T::kBlocks ? scale(sy_read[j]) * scale(sx_read) : scale(sy_read[j]);
        if constexpr (MODE == kScaledE8m0) e8[j] = __builtin_bit_cast(int, sy_read[j]);
      }
    };
    auto read_scales_x = [&](int to, unsigned slot, int i) {
      if constexpr (FLOAT_SCALES && !T::kBlocks) {
        const float *const sxp = reinterpret_cast<const float *>(scales_at(slot)) + wx * TX;
        sx[to] = *reinterpret_cast<const float4_t *>(sxp + i / NT * GROUP_ROWS + g * 4 * NT + i % NT * 4);
      } else if constexpr (MODE == kScaledE8m0) {
        const int *const sxp = reinterpret_cast<const int *>(scales_at(slot)) + wx * TX;
        e8x[to] = sxp[i / NT * GROUP_ROWS + (fr >> 2) * 4 * NT + i % NT * 4 + (fr & 3)];
      }
    };
    auto take_scales_x = [&](int at) {
      if constexpr (FLOAT_SCALES && !T::kBlocks && T::kScaleBytes == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sx[at][e] = scale(sx[at][e]);
      }
    };
    auto read_x = [&](int to, unsigned slot, int i) {
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        const Fragment f = read(slot, x_rows + p * BX * kPieceBytes + i * 16 * kPieceBytes);
        if constexpr (T::kWide) {
          raw_x = f;
        } else {
          x[to][p] = f;
        }
      }
    };
    auto read_y = [&](unsigned slot, int j) {
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        const Fragment f = read(slot, y_rows + p * BY * kPieceBytes + j * 16 * kPieceBytes);
        if constexpr (T::kWide) {
          raw_y[j] = f;
        } else {
          y[p][j] = f;
        }
      }
    };
    // Element `of` (4 JJ of them) of C's sums of step m, with Y's scales (or, a piece later, the ones kept of that step)
    auto add_one = [&](auto step, auto of, bool late) {
      if constexpr (FLOAT_SCALES) {
        constexpr int m = decltype(step)::value, i = m / SPT, h = decltype(of)::value / 4, e = decltype(of)::value % 4;
        constexpr int j = m % SPT * JJ + h;
        const float sy = late ? s_old[m % RING * JJ + h] : s[j];
        if constexpr (e == 0) pin(part[m % RING][h]);
        const float v = part[m % RING][h][e];
        if (T::kBlocks) {
          acc[0][j][i][e] = __builtin_fmaf(v, sy, acc[0][j][i][e]);
        } else {
          acc[0][j][i][e] = __builtin_fmaf(v * sy, sx[i % 2][e], acc[0][j][i][e]);
        }
        if constexpr (e == 3) pin(acc[0][j][i]);
      }
    };
    auto add = [&](auto step, bool late) {
      static_for<4 * JJ>([&](auto of) { add_one(step, of, late); });
    };
    auto products = [&](auto step) {
      constexpr int m = decltype(step)::value, i = m / SPT, j0 = m % SPT * JJ, b = i % 2;
      if constexpr (MODE == kScaledE8m0) {
        acc[0][j0][i] = mfma8<FX, FY>(x[b][0], y[0][j0], acc[0][j0][i], e8x[b], e8[j0]);
      } else if constexpr (T::kWide) {
        // between these products, which take 16 clocks each: what of the step before is added, and of the next X
        // fragment becomes fp16
        static_for<4 * JJ>([&](auto product) {
          constexpr int k = decltype(product)::value, q = k / JJ, h = k % JJ;
          part[m % RING][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[b][0].v[q], y[0][j0 + h].v[q],
                                                                     q == 0 ? zero : part[m % RING][h], 0, 0, 0);
          pin(part[m % RING][h]);
          CCGLIB_PIN;
          if constexpr (m >= LAG) {
            add_one(std::integral_constant<int, m - LAG>{}, product, false);
          } else if constexpr (CARRY) {
            add_one(std::integral_constant<int, m - LAG + STEPS>{}, product, true);
          }
          if constexpr (m % SPT > 0 && k % 2 == 1) {     // (its reads have had a step's time)
            constexpr int WORDS = 8, SLICES = (SPT > 1 ? SPT - 1 : 1) * 4, PER = (WORDS + SLICES - 1) / SLICES, w0 = ((m % SPT - 1) * 4 + k / 2) * PER;
            static_for<PER>([&](auto w) {
              if constexpr (w0 + decltype(w)::value < WORDS) widen_word<FX>(raw_x, x[1 - b][0], w0 + decltype(w)::value);
            });
          }
          CCGLIB_PIN;
        });
      } else if constexpr (T::kScaled) {
        part[m % RING][0] = mfma8<FX, FY>(x[b][0], y[0][j0], zero, 0x7f, 0x7f);
      } else if constexpr (MODE == kHalf) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int h = 0; h < JJ; ++h) acc[0][j0 + h][i] = mfma16(x[b][0], y[0][j0 + h], acc[0][j0 + h][i], q);
        }
      } else {
        constexpr int L = PLANES - 1;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int h = 0; h < JJ; ++h) acc[0][j0 + h][i] = mfma16(x[b][0], y[0][j0 + h], acc[0][j0 + h][i], q);
#pragma unroll
          for (int h = 0; h < JJ; ++h) acc[L][j0 + h][i] = mfma16(x[b][0], y[L][j0 + h], acc[L][j0 + h][i], q);
#pragma unroll
          for (int h = 0; h < JJ; ++h) acc[L][j0 + h][i] = mfma16(x[b][L], y[0][j0 + h], acc[L][j0 + h][i], q);
        }
      }
    };

    unsigned slot = 0, refill = SLOTS - 1;
    if (n >= (unsigned)SLOTS - 1) {   // (SLOTS - 2 later pieces are on their way)
      wait_copies_then_barrier<COPIES * (SLOTS - 2)>();
    } else {
      wait_copies_then_barrier<0>();
    }
    read_scales_y(0);
    take_scales_y();
    read_scales_x(0, 0, 0);
    if constexpr (LAG == 2) take_scales_x(0);
    read_x(0, 0, 0);
    if constexpr (T::kWide) x[0][0] = widened<FX>(raw_x);
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      read_y(0, j);
      if constexpr (T::kWide) y[0][j] = widened<FY>(raw_y[j]);
    }
    if constexpr (FLOAT_SCALES && CARRY) {   // (nothing to add yet)
#pragma unroll
      for (int r = 0; r < RING * JJ; ++r) s_old[r] = 0.f;
#pragma unroll
      for (int r = 0; r < RING; ++r) {
#pragma unroll
        for (int h = 0; h < JJ; ++h) part[r][h] = 0.f;
      }
      if constexpr (!T::kBlocks) sx[1] = 0.f;
    }
    // One piece. REFILL: 0 no further piece is copied; 1 one is, a whole one; 2 one is, perhaps the last, partial one
    auto piece = [&](auto refill_kind) {
      constexpr int REFILL = decltype(refill_kind)::value;
      const unsigned next = slot + 1 == SLOTS ? 0 : slot + 1;
      const typename std::conditional<REFILL == 2, std::true_type, std::false_type>::type end{};
      static_for<STEPS>([&](auto step) {
        constexpr int m = step, i = m / SPT, js = m % SPT, to = (i + 1) % 2;
        constexpr bool at_end = i == NX - 1;
        CCGLIB_PIN;
        if constexpr (COPY_STEPS == 0 && m == 0 && REFILL > 0) static_for<COPIES>([&](auto c) { copy_one(refill, c, end); });
        if constexpr (at_end && js == 0) {
          // (as many later pieces are on their way; behind the last copies all of them have to have arrived)
          constexpr int LATER = REFILL != 0 ? COPIES * (SLOTS - 2) : 0;
          wait_copies_then_barrier<LATER>();
          read_scales_y(next);
        }
        if constexpr (js == 0) {
          read_x(to, at_end ? next : slot, at_end ? 0 : i + 1);
          if constexpr (MODE == kScaledE8m0) read_scales_x(to, at_end ? next : slot, at_end ? 0 : i + 1);
        }
        if constexpr (at_end && T::kWide && js == 0) {
          // (all at once: in turn with what is made of them they cost a round trip through LDS each, 240 against 236 us)
#pragma unroll
          for (int j = 0; j < NY; ++j) read_y(next, j);
        }
#pragma unroll
        for (int h = 0; h < JJ; ++h) pin(y[0][js * JJ + h]);
        products(step);
#pragma unroll
        for (int h = 0; h < JJ; ++h) {
          if constexpr (FLOAT_SCALES) {
            pin(part[m % RING][h]);
          } else {
#pragma unroll
            for (int k = 0; k < T::kSums; ++k) pin(acc[k][js * JJ + h][i]);
          }
        }
        CCGLIB_PIN;
        if constexpr (at_end && !T::kWide) {
#pragma unroll
          for (int h = 0; h < JJ; ++h) read_y(next, js * JJ + h);
        }
        constexpr int c0 = m * PER_STEP < COPIES ? m * PER_STEP : COPIES;
        constexpr int c1 = (m + 1) * PER_STEP < COPIES ? (m + 1) * PER_STEP : COPIES;
        static_assert(c0 == c1 || m < COPY_STEPS, "copies lie in front of the wait");
        if constexpr (c0 < c1 && REFILL > 0) {
          static_for<c1 - c0>([&](auto c) { copy_one(refill, std::integral_constant<int, c0 + decltype(c)::value>{}, end); });
        }
        if constexpr (!T::kWide) {
          if constexpr (m >= LAG) {
            add(std::integral_constant<int, m - LAG>{}, false);
          } else if constexpr (CARRY) {
            add(std::integral_constant<int, m - LAG + STEPS>{}, true);
          }
        }
        if constexpr (FLOAT_SCALES && !T::kBlocks && js == LAG - 1) {
          if constexpr (LAG == 1) take_scales_x(i % 2);
          read_scales_x(to, at_end ? next : slot, at_end ? 0 : i + 1);
        }
        if constexpr (T::kWide) {
          if constexpr (SPT == 1) x[to][0] = widened<FX>(raw_x);
          if constexpr (at_end) {   // (a Y fragment of the next piece, where the last products with its predecessor have been issued)
#pragma unroll
            for (int h = 0; h < JJ; ++h) {
              const int j = js * JJ + h;
              y[0][j] = widened<FY>(raw_y[j]);
            }
          }
        }
      });
      if constexpr (FLOAT_SCALES) {
        if constexpr (CARRY) {
#pragma unroll
          for (int r = 0; r < LAG; ++r) {
#pragma unroll
            for (int h = 0; h < JJ; ++h) {
              const int m = STEPS - LAG + r;
              s_old[m % RING * JJ + h] = s[m % SPT * JJ + h];
            }
          }
        } else {
          static_for<LAG>([&](auto r) { add(std::integral_constant<int, STEPS - LAG + r>{}, false); });
        }
      }
      if constexpr (NX % 2 == 1) {   // (the next piece's first tile, where its predecessor was in use)
#pragma unroll
        for (int p = 0; p < PLANES; ++p) x[0][p] = x[1][p];
        sx[0] = sx[1];
        e8x[0] = e8x[1];
      }
      take_scales_y();
      if constexpr (REFILL > 0) advance();
      refill = slot;
      slot = next;
    };
    // (the piece that K ends in, if it is this block's)
    const unsigned n_whole = (size_t)last * kPieceBytes <= args.k_bytes ? n : n - 1;
    unsigned t = 0;
#pragma unroll 1
    for (; t + SLOTS - 1 < n_whole; ++t) piece(std::integral_constant<int, 1>{});
    if (t + SLOTS - 1 < n) {
      piece(std::integral_constant<int, 2>{});
      ++t;
    }
#pragma unroll 1
    for (; t < n; ++t) piece(std::integral_constant<int, 0>{});
    if constexpr (FLOAT_SCALES && CARRY) {
      static_for<LAG>([&](auto r) { add(std::integral_constant<int, STEPS - LAG + r>{}, true); });
    }
  }

  if constexpr (MODE == kHalfPairs) {
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int i = 0; i < NX; ++i) acc[0][j][i] += acc[T::kSums - 1][j][i] * 0x1p-11f;
    }
  }

  // ---- parts of K joined: in the order of the parts, whichever block arrives last ----
  // The sums go past the L2 of this XCD and are read past the reader's (stores and loads of agent scope), so that no
  // cache has to be written back or emptied: with fences of agent scope in their place one row of 8192 x 8192
  // took 55 us where this takes 17.
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
          const float pair[2] = {acc[0][j][i][2 * h], acc[0][j][i][2 * h + 1]};
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
    const bool is_last = *flag != 0;
    __syncthreads();   // (the epilogue uses the LDS that the flag is in)
    if (!is_last) return;
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
            const unsigned lo = (unsigned)u, hi = (unsigned)(u >> 32);
            if (p == 0) {
              acc[0][j][i][2 * h] = __builtin_bit_cast(float, lo);
              acc[0][j][i][2 * h + 1] = __builtin_bit_cast(float, hi);
            } else {
              acc[0][j][i][2 * h] += __builtin_bit_cast(float, lo);
              acc[0][j][i][2 * h + 1] += __builtin_bit_cast(float, hi);
            }
          }
        }
      }
    }
  }

  // ---- epilogue ----
  const Epilogue epilogue(params);
  constexpr int GROUP_LDS = GROUP_ROWS * kGroupPitch<NY>;
  static_assert(WAVES * GROUP_LDS <= S::kLdsBytes, "the ring holds a group of every wave");
  Group group;
  group.b = at.b;
  group.y = y0 + wy * TY;
  group.lane = lane;
  group.mirror = args.symmetric && at.bx != at.by;
  group.lds = lds + wave * GROUP_LDS;
#pragma unroll
  for (int i = 0; i < NX; i += NT) {
    group.x = x0 + wx * TX + i / NT * GROUP_ROWS;
    float v[NY][4 * NT];
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][4 * t + e] = acc[0][j][i + t][e];
      }
    }
    if (group.y < args.ny && group.x < args.nx) epilogue.store(group, v);
  }
}

}  // namespace real
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_REAL_GEMM_H_
