// C[m][n] (+)= sum over groups g of 128 of K: scale_a[g][m] scale_b[g][n] sum over k in g of A[m][k] B[n][k], 8-bit operands.
//
// B's rows (n, the contiguous axis of C) are X of the product kernel, A's rows Y. With float scales the instruction
// sums one group from zero, and the vector ALU adds it to C's sum with the product of the two scales: one fused operation
// for each element and group where B has a scale for 128 x 128 values (a lane's scale of A times a uniform one), two where
// each row of B has its own. Powers of two (e8m0) are what the matrix instruction takes as its own scales.
// Sums of groups are held in 32 bits and rounded once, to the type of C. Inside a group the 8-bit instruction sums to fewer
// bits, which is enough for a C of 16; a 32-bit C is multiplied by the fp16 instruction (kWide* in real_gemm.h).
#ifndef CCGLIB_AMD_SCALED_GEMM_H_
#define CCGLIB_AMD_SCALED_GEMM_H_

#include "real_gemm.h"
#include "scaled.h"

namespace ccglib_amd {
namespace real {

// Block shapes: BX (columns of C) x BY (rows), waves, ring, waves a SIMD. 128 x 128 comes twice: with four waves, two blocks
// to a unit, and with eight and twice the ring for problems that have no more blocks than units (2048 x 2048 x 4096, float
// scales: 30.5 and 22.2 us; 4096 x 2048 x 2048, two blocks a unit: 22.1 and 25.3). 192 x 192 fills units that larger blocks
// would leave idle and smaller ones would not feed (3000 x 3000 x 8192, e8m0: 256 x 256 78 us, 192 x 192 62, 128 x 128 101;
// float scales of rows 111, 84, 127).
#define CCGLIB_SCALED_SHAPES(DO) \
  DO(0, 256, 256, 2, 4, 2, 2)    \
  DO(1, 128, 128, 2, 2, 2, 2)    \
  DO(2, 64, 64, 2, 2, 4, 2)      \
  DO(3, 64, 32, 4, 1, 6, 2)      \
  DO(4, 128, 128, 4, 2, 4, 2)    \
  DO(5, 192, 192, 2, 4, 3, 2)
// (fp16 operands take twice the registers)
#define CCGLIB_WIDE_SHAPES(DO) \
  DO(0, 128, 256, 2, 4, 2, 2)  \
  DO(1, 128, 128, 2, 2, 2, 2)  \
  DO(2, 64, 64, 2, 2, 4, 2)    \
  DO(3, 64, 32, 4, 1, 6, 2)    \
  DO(4, 128, 128, 4, 2, 4, 2)

struct StoreC {
  struct Params {
    char *c;
    size_t pitch, batch;     // elements from row to row, from matrix to matrix
    unsigned nx, ny;
    int type, accumulate;
  };
  const Params &p;
  __device__ explicit StoreC(const Params &params) : p(params) {}

  template <int NY, int N> __device__ __forceinline__ void store(const Group &g, float (&v)[NY][N]) const {
    const unsigned x = g.x + (g.lane >> 4) * N, left = x < p.nx ? p.nx - x : 0;
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      const unsigned y = g.y + j * 16 + (g.lane & 15);
      if (y >= p.ny || left == 0) continue;
      const size_t at = (size_t)g.b * p.batch + (size_t)y * p.pitch + x;
      if (p.accumulate) {   // (32-bit C)
        float *const c = reinterpret_cast<float *>(p.c) + at;
#pragma unroll
        for (int e = 0; e < N; ++e) v[j][e] += (unsigned)e < left ? c[e] : 0.f;
        store_row(c, left, v[j]);
      } else if (p.type == kFloat32) {
        store_row(reinterpret_cast<float *>(p.c) + at, left, v[j]);
      } else if (p.type == kFloat16) {
        store_row(reinterpret_cast<_Float16 *>(p.c) + at, left, v[j]);
      } else {
        store_row(reinterpret_cast<__bf16 *>(p.c) + at, left, v[j]);
      }
    }
  }
};

template <int MODE> hipError_t launch_scaled_mode(const ScaledGemmParams &p, const Args &a, hipStream_t stream);
template <> hipError_t launch_scaled_mode<kScaledBlocks>(const ScaledGemmParams &p, const Args &a, hipStream_t stream);
template <> hipError_t launch_scaled_mode<kScaledRows>(const ScaledGemmParams &p, const Args &a, hipStream_t stream);
template <> hipError_t launch_scaled_mode<kScaledE8m0>(const ScaledGemmParams &p, const Args &a, hipStream_t stream);
template <> hipError_t launch_scaled_mode<kWideBlocks>(const ScaledGemmParams &p, const Args &a, hipStream_t stream);
template <> hipError_t launch_scaled_mode<kWideRows>(const ScaledGemmParams &p, const Args &a, hipStream_t stream);
template <> hipError_t launch_scaled_mode<kWideE8m0>(const ScaledGemmParams &p, const Args &a, hipStream_t stream);

#ifdef CCGLIB_SCALED_MODE
template <int MODE, int FX, int FY>
hipError_t launch_scaled(int shape, unsigned grid, const Args &a, const StoreC::Params &e, hipStream_t stream) {
#define CCGLIB_CASE(ID, BX, BY, WX, WY, SLOTS, EU)                                                       \
  case ID:                                                                                                 \
    if constexpr (!ModeTraits<MODE>::kBlocks || BX % 128 == 0 || 128 % BX == 0) {                          \
      gemm_real<MODE, FX, FY, BX, BY, WX, WY, SLOTS, EU, StoreC><<<grid, 64 * WX * WY, 0, stream>>>(a, e); \
    }                                                                                                      \
    break;
  if constexpr (ModeTraits<MODE>::kWide) {
    switch (shape) { CCGLIB_WIDE_SHAPES(CCGLIB_CASE) }
  } else {
    switch (shape) { CCGLIB_SCALED_SHAPES(CCGLIB_CASE) }
  }
#undef CCGLIB_CASE
  return hipGetLastError();
}

template <> hipError_t launch_scaled_mode<CCGLIB_SCALED_MODE>(const ScaledGemmParams &p, const Args &a, hipStream_t stream) {
  constexpr int MODE = CCGLIB_SCALED_MODE;
  StoreC::Params e;
  e.c = static_cast<char *>(p.c);
  e.pitch = p.pitch_c;
  e.batch = (size_t)p.m * p.pitch_c;
  e.nx = p.n;
  e.ny = p.m;
  e.type = p.type_c;
  e.accumulate = p.accumulate;
  const unsigned grid = a.batch * a.parts * a.blocks_x * a.blocks_y;
  const bool a4 = p.type_a == kFloat8e4m3, b4 = p.type_b == kFloat8e4m3;
  if (a4 && b4) return launch_scaled<MODE, 0, 0>(p.plan.shape, grid, a, e, stream);
  if (b4) return launch_scaled<MODE, 0, 1>(p.plan.shape, grid, a, e, stream);
  if (a4) return launch_scaled<MODE, 1, 0>(p.plan.shape, grid, a, e, stream);
  return launch_scaled<MODE, 1, 1>(p.plan.shape, grid, a, e, stream);
}
#endif

}  // namespace real
}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_SCALED_GEMM_H_
