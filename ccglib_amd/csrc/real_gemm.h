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
#ifndef CCGLIB_AMD_REAL_GEMM_H_
#define CCGLIB_AMD_REAL_GEMM_H_

#include <type_traits>

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

struct Fragment {
  int4_t v[2];
};

__device__ __forceinline__ int8x_t joined(const Fragment &f) {
  return int8x_t{f.v[0][0], f.v[0][1], f.v[0][2], f.v[0][3], f.v[1][0], f.v[1][1], f.v[1][2], f.v[1][3]};
}

// FX, FY: format codes of 8-bit operands (0 e4m3, 1 e5m2)
template <int FX, int FY>
__device__ __forceinline__ float4_t mfma8(const Fragment &x, const Fragment &y, float4_t c, int sx, int sy) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(joined(x), joined(y), c, FX, FY, 0, sx, 0, sy);
}
// A lane's 32 values of 8 bits as fp16, four operands of the fp16 instruction
struct WideFragment {
  half8_t v[4];
};
template <int FORMAT> __device__ __forceinline__ WideFragment widened(const Fragment &f) {
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  WideFragment r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const unsigned word = (unsigned)f.v[q / 2][q % 2 * 2 + w];
      half2_t lo, hi;
      if constexpr (FORMAT == 0) {
        lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, true);
      } else {   // (e5m2 is the upper half of fp16)
        lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(word, word, 0x010c000cu));
        hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(word, word, 0x030c020cu));
      }
      r.v[q][4 * w] = lo[0];
      r.v[q][4 * w + 1] = lo[1];
      r.v[q][4 * w + 2] = hi[0];
      r.v[q][4 * w + 3] = hi[1];
    }
  }
  return r;
}
__device__ __forceinline__ float4_t mfma_wide(const WideFragment &x, const WideFragment &y, float4_t c) {
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v[q], y.v[q], c, 0, 0, 0);
  return c;
}
// 2^(byte - 127); 255 stands for NaN
__device__ __forceinline__ float power_of_two(unsigned byte) {
  const float p = __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte << 23);
  return byte == 255 ? __builtin_nanf("") : p;
}

__device__ __forceinline__ float4_t mfma16(const Fragment &x, const Fragment &y, float4_t c) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, x.v[s]), __builtin_bit_cast(half8_t, y.v[s]),
                                               c, 0, 0, 0);
  }
  return c;
}

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

// Epilogue: has `Params`, a constructor from them, and
//   template <int N> void store(unsigned b, unsigned y, unsigned x, const float (&v)[N], bool mirror)
// for N consecutive x of row y (which may lie beyond D); mirror: D[x][y] is wanted as well.
template <int MODE, int FX, int FY, int BX, int BY, int WX, int WY, int SLOTS, int WAVES_PER_EU, class Epilogue>
__global__ __launch_bounds__(64 * WX * WY, WAVES_PER_EU) void gemm_real(Args args, typename Epilogue::Params params) {
  using S = Shape<MODE, BX, BY, WX, WY, SLOTS>;
  using T = ModeTraits<MODE>;
  constexpr int WAVES = WX * WY, PLANES = T::kPlanes;
  constexpr int TX = BX / WX, TY = BY / WY, NX = TX / 16, NY = TY / 16;
  constexpr int NT = NX < 4 ? NX : 4, GROUP_ROWS = 16 * NT;
  constexpr int X_COPIES = BX / 8 * PLANES, COPIES_ALL = X_COPIES + BY / 8 * PLANES;
  constexpr int OPERAND_COPIES = COPIES_ALL / WAVES;
  constexpr int SCALE_COPIES = T::kScaled ? (BX + BY + 63) / 64 : 0;
  constexpr int COPIES = OPERAND_COPIES + (T::kScaled ? 1 : 0);
  static_assert(COPIES_ALL % WAVES == 0 && SCALE_COPIES <= WAVES && NX % NT == 0, "shape");
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
    int q = wave + n * WAVES;
    const bool of_x = q < X_COPIES;
    if (!of_x) q -= X_COPIES;
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
  auto copy = [&](unsigned piece, unsigned slot) {
    const unsigned to = lds_base + slot * S::kSlotBytes;
    const size_t k = (size_t)piece * kPieceBytes;
    const bool whole = (piece + 1) * (unsigned)kPieceBytes <= args.k_bytes;
#pragma unroll
    for (int n = 0; n < OPERAND_COPIES; ++n) {
      const int q = wave + n * WAVES;
      const bool of_x = q < X_COPIES;
      const int plane = PLANES == 1 ? 0 : of_x ? q / (BX / 8) : (q - X_COPIES) / (BY / 8);
      const char *from = (of_x ? x_base : y_base) + k;
      if (PLANES > 1 && plane) from += of_x ? args.x_plane : args.y_plane;
      if (whole) {
        load_1k_to_lds(from, offset[n], to + q * 1024);
      } else {
        load_1k_to_lds_by_lane(k + chunk * 16 < args.k_bytes ? from + offset[n] : g_zeros, to + q * 1024);
      }
    }
    if constexpr (T::kScaled) {
      const size_t s = (size_t)piece * scale_step;
      if constexpr (BX % 64 == 0) {
        load_scales_to_lds<T::kScaleBytes>(scale_base + s, scale_offset, to + S::kXBytes + S::kYBytes + scale_lds);
      }
    }
  };
  static_assert(!T::kScaled || BX % 64 == 0, "scales of X fill whole copies");

  // ---- fragments ----
  const int fr = lane & 15, g = lane >> 4;
  const unsigned frag0 = fr * kPieceBytes + ((g ^ (fr & 7)) << 4), frag1 = fr * kPieceBytes + (((g + 4) ^ (fr & 7)) << 4);
  auto read = [&](unsigned slot, int from) {
    const char *p = lds + slot * S::kSlotBytes + from;
    Fragment f;
    f.v[0] = *reinterpret_cast<const int4_t *>(p + frag0);
    f.v[1] = *reinterpret_cast<const int4_t *>(p + frag1);
    return f;
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

  auto multiply = [&](unsigned slot) {
    Fragment y[PLANES][NY];
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
#pragma unroll
      for (int j = 0; j < NY; ++j) y[p][j] = read(slot, y_rows + p * BY * kPieceBytes + j * 16 * kPieceBytes);
    }
    const char *scales = lds + slot * S::kSlotBytes + S::kXBytes + S::kYBytes;
    if constexpr (T::kScaled && MODE != kScaledE8m0) {
      const float *const sx = reinterpret_cast<const float *>(scales) + wx * TX;
      const float *const sy = reinterpret_cast<const float *>(scales) + BX + wy * TY;
      auto scale = [](float stored) {
        return T::kScaleBytes == 1 ? power_of_two(__builtin_bit_cast(unsigned, stored)) : stored;
      };
      float s[NY];
      typename std::conditional<T::kWide, WideFragment, int>::type y16[NY];
#pragma unroll
      for (int j = 0; j < NY; ++j) {
        s[j] = scale(sy[j * 16 + fr]);
        if (T::kBlocks) s[j] *= scale(sx[0]);
        if constexpr (T::kWide) y16[j] = widened<FY>(y[0][j]);
      }
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const Fragment x = read(slot, x_rows + i * 16 * kPieceBytes);
        typename std::conditional<T::kWide, WideFragment, int>::type x16;
        if constexpr (T::kWide) x16 = widened<FX>(x);
        float4_t sx4 = zero;
        if (!T::kBlocks) {
          sx4 = *reinterpret_cast<const float4_t *>(sx + i / NT * GROUP_ROWS + g * 4 * NT + i % NT * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) sx4[e] = scale(sx4[e]);
        }
#pragma unroll
        for (int j = 0; j < NY; ++j) {
          float4_t part;
          if constexpr (T::kWide) {
            part = mfma_wide(x16, y16[j], zero);
          } else {
            part = mfma8<FX, FY>(x, y[0][j], zero, 0x7f, 0x7f);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (T::kBlocks) {
              acc[0][j][i][e] = __builtin_fmaf(part[e], s[j], acc[0][j][i][e]);
            } else {
              acc[0][j][i][e] = __builtin_fmaf(part[e] * s[j], sx4[e], acc[0][j][i][e]);
            }
          }
        }
      }
    } else if constexpr (MODE == kScaledE8m0) {
      const int *const sx = reinterpret_cast<const int *>(scales) + wx * TX;
      const int *const sy = reinterpret_cast<const int *>(scales) + BX + wy * TY;
      int s[NY];
#pragma unroll
      for (int j = 0; j < NY; ++j) s[j] = sy[j * 16 + fr];
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const Fragment x = read(slot, x_rows + i * 16 * kPieceBytes);
        const int t = sx[i / NT * GROUP_ROWS + (fr >> 2) * 4 * NT + i % NT * 4 + (fr & 3)];
#pragma unroll
        for (int j = 0; j < NY; ++j) acc[0][j][i] = mfma8<FX, FY>(x, y[0][j], acc[0][j][i], t, s[j]);
      }
    } else if constexpr (MODE == kHalf) {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const Fragment x = read(slot, x_rows + i * 16 * kPieceBytes);
#pragma unroll
        for (int j = 0; j < NY; ++j) acc[0][j][i] = mfma16(x, y[0][j], acc[0][j][i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const Fragment xh = read(slot, x_rows + i * 16 * kPieceBytes);
        const Fragment xl = read(slot, x_rows + BX * kPieceBytes + i * 16 * kPieceBytes);
#pragma unroll
        for (int j = 0; j < NY; ++j) {
          acc[0][j][i] = mfma16(xh, y[0][j], acc[0][j][i]);
          acc[T::kSums - 1][j][i] = mfma16(xh, y[PLANES - 1][j], acc[T::kSums - 1][j][i]);
          acc[T::kSums - 1][j][i] = mfma16(xl, y[0][j], acc[T::kSums - 1][j][i]);
        }
      }
    }
  };

  // ---- K loop ----
  const unsigned n = last > first ? last - first : 0;
#pragma unroll
  for (int t = 0; t < SLOTS - 1; ++t) {
    if ((unsigned)t < n) copy(first + t, t);
  }
  unsigned slot = 0, refill = SLOTS - 1;
#pragma unroll 1
  for (unsigned t = 0; t < n; ++t) {
    if (t + SLOTS - 1 < n + (SLOTS > 2 ? 1 : 0)) {   // (SLOTS - 2 later pieces are on their way)
      wait_copies_then_barrier<COPIES * (SLOTS - 2)>();
    } else {
      wait_copies_then_barrier<0>();
    }
    if (t + SLOTS - 1 < n) copy(first + t + SLOTS - 1, refill);
    multiply(slot);
    refill = slot;
    slot = slot + 1 == SLOTS ? 0 : slot + 1;
  }

  if constexpr (MODE == kHalfPairs) {
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int i = 0; i < NX; ++i) acc[0][j][i] += acc[T::kSums - 1][j][i] * 0x1p-11f;
    }
  }

  // ---- pieces of K joined: in the order of the pieces, whichever block arrives last ----
  if (args.parts > 1) {
    constexpr size_t BLOCK = (size_t)BX * BY;   // floats
    float4_t *const mine = reinterpret_cast<float4_t *>(args.partial + ((size_t)at.tile * args.parts + at.part) * BLOCK);
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int i = 0; i < NX; ++i) mine[(j * NX + i) * (64 * WAVES) + threadIdx.x] = acc[0][j][i];
    }
    __threadfence();
    __syncthreads();
    unsigned *const flag = reinterpret_cast<unsigned *>(lds);
    if (threadIdx.x == 0) {
      const unsigned before = __hip_atomic_fetch_add(args.arrived + at.tile, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
      *flag = before + 1 == args.parts;
      if (before + 1 == args.parts) {
        __hip_atomic_store(args.arrived + at.tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    __syncthreads();
    if (!*flag) return;
    __threadfence();
    const float4_t *from = reinterpret_cast<const float4_t *>(args.partial + (size_t)at.tile * args.parts * BLOCK);
#pragma unroll
    for (int j = 0; j < NY; ++j) {
#pragma unroll
      for (int i = 0; i < NX; ++i) acc[0][j][i] = from[(j * NX + i) * (64 * WAVES) + threadIdx.x];
    }
#pragma unroll 1
    for (unsigned p = 1; p < args.parts; ++p) {
      from += BLOCK / 4;
#pragma unroll
      for (int j = 0; j < NY; ++j) {
#pragma unroll
        for (int i = 0; i < NX; ++i) acc[0][j][i] += from[(j * NX + i) * (64 * WAVES) + threadIdx.x];
      }
    }
  }

  // ---- epilogue ----
  const Epilogue epilogue(params);
  const bool mirror = args.symmetric && at.bx != at.by;
#pragma unroll
  for (int j = 0; j < NY; ++j) {
    const unsigned y = y0 + wy * TY + j * 16 + fr;
#pragma unroll
    for (int i = 0; i < NX; i += NT) {
      const unsigned x = x0 + wx * TX + i / NT * GROUP_ROWS + g * 4 * NT;
      float v[4 * NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * t + e] = acc[0][j][i + t][e];
      }
      if (y < args.ny && x < args.nx) epilogue.template store<4 * NT>(at.b, y, x, v, mirror);
    }
  }
}

}  // namespace real
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_REAL_GEMM_H_
