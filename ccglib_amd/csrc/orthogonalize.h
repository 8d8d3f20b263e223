// Kernels of the orthogonalised updates that multiply: X X^T, b A + c A A, a X + P X (see orthogonalize.hip).
#ifndef CCGLIB_AMD_ORTHOGONALIZE_H_
#define CCGLIB_AMD_ORTHOGONALIZE_H_

#include "real_gemm.h"
#include "scaled.h"

namespace ccglib_amd {
namespace real {

// Matrices of the chain: fp16, or two fp16 for each value (v = first + second * 2^-11), a plane each.
template <bool PAIRS> struct Halves {
  static __device__ __forceinline__ float get(const _Float16 *p, size_t at, size_t plane) {
    const float h = (float)p[at];
    return PAIRS ? __builtin_fmaf((float)p[at + plane], 0x1p-11f, h) : h;
  }
  static __device__ __forceinline__ void put(_Float16 *p, size_t at, size_t plane, float v) {
    const _Float16 h = (_Float16)v;
    p[at] = h;
    if (PAIRS) p[at + plane] = (_Float16)((v - (float)h) * 0x1p11f);
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

  template <int N>
  __device__ __forceinline__ void store(unsigned b, unsigned y, unsigned x, const float (&v)[N], bool mirror) const {
    using H = Halves<PAIRS>;
    const float f = p.factor ? p.factor[b] : 1.f;
    const unsigned left = p.nx - x;
    float *const diagonal = p.diagonal + (size_t)b * p.diagonal_pitch;
    float *const diagonal_p = p.diagonal_p + (size_t)b * p.diagonal_pitch;
    const _Float16 *const old = p.old + (size_t)b * p.old_batch + (size_t)y * p.old_pitch + x;
    float w[N];
    if constexpr (STEP == kGram) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        w[e] = f * f * v[e];
        if (x + e == y) {
          diagonal[y] = w[e];
          w[e] = 0.f;
        }
      }
    } else if constexpr (STEP == kSquare) {
      const float dy = diagonal[y];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if ((unsigned)e < left) {
          if (x + e == y) {
            diagonal_p[y] = __builtin_fmaf(p.c, __builtin_fmaf(dy, dy, v[e]), p.b * dy);
            w[e] = 0.f;
          } else {
            const float o = H::get(old, e, p.old_plane);
            w[e] = __builtin_fmaf(p.c, __builtin_fmaf(dy + diagonal[x + e], o, v[e]), p.b * o);
          }
        }
      }
    } else {
      const float dy = STEP == kUpdate ? p.a + diagonal_p[y] : 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if ((unsigned)e < left) {
          const float d = STEP == kUpdate ? dy : p.a + diagonal_p[x + e];
          w[e] = f * __builtin_fmaf(d, H::get(old, e, p.old_plane), v[e]);
        }
      }
      if (p.out) {
        const size_t at = (size_t)b * p.out_batch + (size_t)y * p.out_pitch + x;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if ((unsigned)e < left) {
            if (p.out_type == kFloat32) {
              static_cast<float *>(p.out)[at + e] = w[e];
            } else if (p.out_type == kFloat16) {
              static_cast<_Float16 *>(p.out)[at + e] = (_Float16)w[e];
            } else {
              static_cast<__bf16 *>(p.out)[at + e] = (__bf16)w[e];
            }
          }
        }
        return;
      }
    }
    _Float16 *const to = p.to + (size_t)b * p.to_batch;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if ((unsigned)e < left) H::put(to, (size_t)y * p.to_pitch + x + e, p.to_plane, w[e]);
    }
    if (STEP == kUpdate || mirror) {
      _Float16 *const t = STEP == kUpdate ? p.to_t + (size_t)b * p.to_t_batch : to;
      const unsigned pitch = STEP == kUpdate ? p.to_t_pitch : p.to_pitch;
      const size_t plane = STEP == kUpdate ? p.to_t_plane : p.to_plane;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if ((unsigned)e < left) H::put(t, (size_t)(x + e) * pitch + y, plane, w[e]);
      }
    }
  }
};

#define CCGLIB_HALF_SHAPES(DO) \
  DO(0, 256, 256, 2, 4, 2, 2)  \
  DO(1, 128, 128, 2, 2, 2, 2)  \
  DO(2, 64, 64, 2, 2, 4, 2)
#define CCGLIB_HALF_PAIRS_SHAPES(DO) \
  DO(0, 128, 128, 2, 4, 2, 2)        \
  DO(1, 64, 64, 2, 2, 2, 2)

struct HalfShape {
  unsigned bx, by;
};

}  // namespace real
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_ORTHOGONALIZE_H_
