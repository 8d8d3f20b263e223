// Kernels of the orthogonalised updates that multiply: X X^T, b A + c A A, a X + P X (see orthogonalize.hip).
#ifndef CCGLIB_AMD_ORTHOGONALIZE_H_
#define CCGLIB_AMD_ORTHOGONALIZE_H_

#include "real_gemm.h"
#include "scaled.h"

namespace ccglib_amd {
namespace real {

// Matrices of the chain: fp16, or two fp16 for each value (v = first + second * 2^-11), a plane each. Rows are padded to a
// whole 128 bytes, with zeros.
template <bool PAIRS> struct Halves {
  // (of two parts both see v rounded to 32 bits: made of the operations behind v in one instruction, the first part would
  // now and then be the next one of fp16, and the second one what is left of another)
  static __device__ __forceinline__ _Float16 part(float v, int plane) {
    if constexpr (PAIRS) asm("" : "+v"(v));
    const _Float16 h = (_Float16)v;
    return plane == 0 ? h : (_Float16)((v - (float)h) * 0x1p11f);
  }
  static __device__ __forceinline__ void put(_Float16 *p, size_t plane, float v) {
    p[0] = part(v, 0);
    if (PAIRS) p[plane] = part(v, 1);
  }
  // N (4 or 8) neighbours, at a multiple of N
  template <int N> static __device__ __forceinline__ void load(const _Float16 *p, size_t plane, float (&v)[N]) {
    constexpr int E = N < 8 ? N : 8;
    typedef _Float16 piece_t __attribute__((ext_vector_type(E)));
#pragma unroll
    for (int i = 0; i < N; i += E) {
      const piece_t h = *reinterpret_cast<const piece_t *>(p + i);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i + e] = (float)h[e];
      if constexpr (PAIRS) {
        const piece_t l = *reinterpret_cast<const piece_t *>(p + plane + i);
#pragma unroll
        for (int e = 0; e < E; ++e) v[i + e] = __builtin_fmaf((float)l[e], 0x1p-11f, v[i + e]);
      }
    }
  }
  template <int N> static __device__ __forceinline__ void store(_Float16 *p, size_t plane, const float (&v)[N]) {
    constexpr int E = N < 8 ? N : 8;
    typedef _Float16 piece_t __attribute__((ext_vector_type(E)));
#pragma unroll
    for (int k = 0; k < (PAIRS ? 2 : 1); ++k) {
#pragma unroll
      for (int i = 0; i < N; i += E) {
        piece_t w;
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = part(v[i + e], k);
        *reinterpret_cast<piece_t *>(p + k * plane + i) = w;
      }
    }
  }
};

// What becomes of a product's sums v:
//   kGram    A = f^2 v
//   kSquare  P = b A + c A A, v = E E with A = D + E: off the diagonal b E + c ((d[y] + d[x]) E + v), on it b d + c (d^2 + v)
//   kUpdate  X = f ((a + p[y]) X + v), v = (P - diag p) X; both orientations, or the result in the caller's type
//   kUpdateT the same of X^T: (a + p[x])
// A and P are kept as their diagonals, in 32 bits, and the rest, whose values are smaller: late steps have A near the
// unit matrix and P near a multiple of it, and rounding those diagonals to fp16 was half of the result's error
// (0.0014 to 0.0009 of |X|, simulated for 96 x 128 to 512 x 2048).
enum ChainStep { kGram, kSquare, kUpdate, kUpdateT };

template <bool PAIRS, int STEP> struct StoreChain {
  struct Params {
    _Float16 *to, *to_t;            // to_t: X^T (kUpdate)
    const _Float16 *old;            // A, X or X^T
    void *out;                      // the last product of all: the caller's matrix, instead of `to`
    const float *factor;            // [batch], null: 1
    float *diagonal;                // [batch][diagonal_pitch]: of A (kGram writes, kSquare reads), of P (kSquare writes, kUpdate reads)
    float *diagonal_p;
    size_t to_batch, to_t_batch, old_batch, out_batch;           // elements
    size_t to_plane, to_t_plane, old_plane;
    unsigned to_pitch, to_t_pitch, old_pitch, diagonal_pitch;
    size_t out_pitch;
    unsigned nx, ny;
    float a, b, c;
    int out_type;
  };
  const Params &p;
  __device__ explicit StoreChain(const Params &params) : p(params) {}

  // The group's transpose, through LDS into rows of whole pieces of 16 bytes: two lanes with neighbouring y exchange the other's
  // half of each pair of x, so that LDS is written 4 bytes at a time.
  template <int NY, int N>
  __device__ __forceinline__ void store_transposed(const Group &g, const float (&v)[NY][N], _Float16 *t, size_t pitch, size_t plane) const {
    using H = Halves<PAIRS>;
    constexpr int PITCH = kGroupPitch<NY>, CHUNKS = NY * 2;      // pieces of a row
    const int fr = g.lane & 15;
    const bool odd = fr & 1;
#pragma unroll
    for (int k = 0; k < (PAIRS ? 2 : 1); ++k) {
#pragma unroll
      for (int j = 0; j < NY; ++j) {
        const bool inside = g.y + j * 16 + fr < p.ny;           // (behind the rows' end: zeros)
        char *const to = g.lds + ((g.lane >> 4) * N + odd) * PITCH + (j * 16 + (fr & ~1)) * 2;
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
          const half2_t two = {H::part(v[j][e], k), H::part(v[j][e + 1], k)};
          const unsigned mine = inside ? __builtin_bit_cast(unsigned, two) : 0u;
          const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)mine, 0xb1, 0xf, 0xf, true);   // lane ^ 1
          // even y: x = e of both; odd y: x = e + 1 of both
          *reinterpret_cast<unsigned *>(to + e * PITCH) = __builtin_amdgcn_perm(mine, other, odd ? 0x07060302u : 0x01000504u);
        }
      }
#pragma unroll
      for (int r = 0; r < 4 * N * CHUNKS / 64; ++r) {
        const int at = r * 64 + g.lane, row = at / CHUNKS, chunk = at % CHUNKS;
        const int4_t piece = *reinterpret_cast<const int4_t *>(g.lds + row * PITCH + chunk * 16);
        const unsigned x = g.x + row, y = g.y + chunk * 8;
        if (x < p.nx && y < p.ny) *reinterpret_cast<int4_t *>(t + k * plane + (size_t)x * pitch + y) = piece;
      }
    }
  }

  template <int NY, int N> __device__ __forceinline__ void store(const Group &g, float (&v)[NY][N]) const {
    using H = Halves<PAIRS>;
    const float f = p.factor ? p.factor[g.b] : 1.f;
    const unsigned x = g.x + (g.lane >> 4) * N, left = x < p.nx ? p.nx - x : 0;
    float *const diagonal = p.diagonal + (size_t)g.b * p.diagonal_pitch;
    float *const diagonal_p = p.diagonal_p + (size_t)g.b * p.diagonal_pitch;
    float dx[N];           // of the columns; (rows of diagonals are as long as rows of A, and zero behind their end)
    if constexpr (STEP == kSquare || STEP == kUpdateT) {
      const float *const d = (STEP == kSquare ? diagonal : diagonal_p) + x;
#pragma unroll
      for (int e = 0; e < N; ++e) dx[e] = left > 0 ? d[e] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      const unsigned y = g.y + j * 16 + (g.lane & 15);
      float(&w)[N] = v[j];
      if (y >= p.ny || left == 0) continue;
      float old[N];
      if constexpr (STEP != kGram) H::load(p.old + (size_t)g.b * p.old_batch + (size_t)y * p.old_pitch + x, p.old_plane, old);
      if constexpr (STEP == kGram) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          w[e] *= f * f;
          if (x + e == y) {
            diagonal[y] = w[e];
            w[e] = 0.f;
          }
        }
      } else if constexpr (STEP == kSquare) {
        const float dy = diagonal[y];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (x + e == y) {
            diagonal_p[y] = __builtin_fmaf(p.c, __builtin_fmaf(dy, dy, w[e]), p.b * dy);
            w[e] = 0.f;
          } else {
            w[e] = __builtin_fmaf(p.c, __builtin_fmaf(dy + dx[e], old[e], w[e]), p.b * old[e]);
          }
        }
      } else {
        const float dy = STEP == kUpdate ? diagonal_p[y] : 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = f * __builtin_fmaf(p.a + (STEP == kUpdate ? dy : dx[e]), old[e], w[e]);
        if (STEP == kUpdateT || p.out) {
          const size_t at = (size_t)g.b * p.out_batch + (size_t)y * p.out_pitch + x;
          if (p.out_type == kFloat32) {
            store_row(static_cast<float *>(p.out) + at, left, w);
          } else if (p.out_type == kFloat16) {
            store_row(static_cast<_Float16 *>(p.out) + at, left, w);
          } else {
            store_row(static_cast<__bf16 *>(p.out) + at, left, w);
          }
          continue;
        }
      }
      if (left < (unsigned)N) {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = (unsigned)e < left ? w[e] : 0.f;
      }
      H::store(p.to + (size_t)g.b * p.to_batch + (size_t)y * p.to_pitch + x, p.to_plane, w);
    }
    if constexpr (STEP == kUpdate) {
      if (!p.out) store_transposed(g, v, p.to_t + (size_t)g.b * p.to_t_batch, p.to_t_pitch, p.to_t_plane);
    } else if constexpr (STEP != kUpdateT) {
      if (g.mirror) store_transposed(g, v, p.to + (size_t)g.b * p.to_batch, p.to_pitch, p.to_plane);
    }
  }
};

// Block shapes: BX x BY, waves, ring, waves a SIMD. 128 x 128 with eight waves is for products that have no more blocks than
// units: P X of 1024 x 4096 takes 22.2 us with four waves a block and 15.6 with eight.
// 192 x 192: A of 4096 x 8192 has 136 blocks of 256 x 256 for 256 units and takes 167 us, with 253 blocks 136.
#define CCGLIB_HALF_SHAPES(DO) \
  DO(0, 256, 256, 2, 4, 2, 2)  \
  DO(1, 128, 128, 2, 2, 2, 2)  \
  DO(2, 64, 64, 2, 2, 4, 2)    \
  DO(3, 128, 128, 4, 2, 4, 2)  \
  DO(4, 192, 192, 4, 2, 3, 2)
#define CCGLIB_HALF_PAIRS_SHAPES(DO) \
  DO(0, 128, 128, 2, 4, 2, 2)        \
  DO(1, 64, 64, 2, 2, 2, 2)

}  // namespace real
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_ORTHOGONALIZE_H_
