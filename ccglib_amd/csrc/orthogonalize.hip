// Orthogonalised updates: X0 = G / (|G| + epsilon) (G^T where that is the wider one), |.| the Frobenius norm, then steps of
//   A = X X^T,  P = b A + c A A,  X <- a X + P X,
// which drive every singular value of X towards 1 (a Newton-Schulz iteration of degree five).
//
// All three products run on gemm_real. A and P are symmetric: blocks below the diagonal are multiplied, and stored twice;
// their diagonals are kept apart, in 32 bits.
// P X needs X with its columns contiguous, so X is kept in both orientations, and the epilogue of P X writes both.
//
// bf16 updates: the chain is fp16 (11 bits where the update has 8), sums are 32 bits. X0 is G times a power of two, which
// loses nothing of values above 2^-24 |G|, and 2^-32 |G| at most of those below, which have fewer bits in fp16; the rest of
// 1 / (|G| + epsilon) is a factor of the first step's epilogues. fp16 and fp32 updates: every
// value of the chain is two fp16, 22 bits, and three of the four products are added up (the fourth is 2^-22 of the first).
// |G| is summed in 64 bits, so that no G overflows it.
#include <algorithm>

#include "orthogonalize.h"
#include "real_plan.h"

namespace ccglib_amd {
namespace {

constexpr size_t kAlign = 256;
size_t up(size_t n, size_t to) { return ceil_div(n, to) * to; }

// Whether a value of the chain is two fp16.
bool as_pairs(int type) { return type != kBfloat16; }

#define HIP_PASS(expr)                         \
  do {                                         \
    const hipError_t e_ = (expr);              \
    if (e_ != hipSuccess) return e_;           \
  } while (0)

template <int TYPE> struct Value;
template <> struct Value<kFloat32> { using type = float; };
template <> struct Value<kFloat16> { using type = _Float16; };
template <> struct Value<kBfloat16> { using type = __bf16; };

// partial[b][block] = sum of the squares of a part of matrix b: a block has `rows` x kNormColumns values, a thread eight
// neighbours at a time. Bound by memory: 4096 x 8192 bf16 15 us, 4.5 TB/s; 4096 x 1024 5 us, two round trips.
constexpr unsigned kNormColumns = 2048;
template <int TYPE>
__global__ __launch_bounds__(256) void sum_of_squares(const typename Value<TYPE>::type *in, size_t pitch, unsigned m, unsigned n,
                                                      unsigned rows, double *partial) {
  using V = typename Value<TYPE>::type;
  typedef V eight_t __attribute__((ext_vector_type(8), aligned(sizeof(V))));
  const unsigned b = blockIdx.z, c = blockIdx.x * kNormColumns + threadIdx.x * 8, r0 = blockIdx.y * rows;
  const V *g = in + ((size_t)b * m + r0) * pitch + c;
  double sum = 0.0;
  if (c + 8 <= n) {
#pragma unroll 8
    for (unsigned r = 0; r < rows; ++r) {
      if (r0 + r >= m) break;
      const eight_t v = *reinterpret_cast<const eight_t *>(g + (size_t)r * pitch);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double d = (double)(float)v[e];
        sum = __builtin_fma(d, d, sum);
      }
    }
  } else if (c < n) {
    for (unsigned r = 0; r < rows && r0 + r < m; ++r) {
      for (unsigned e = 0; c + e < n; ++e) {
        const double d = (double)(float)g[(size_t)r * pitch + e];
        sum = __builtin_fma(d, d, sum);
      }
    }
  }
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  __shared__ double waves[4];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    partial[((size_t)b * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
  }
}

// The sum of `count` partial sums, by 256 threads, in all of them.
__device__ __forceinline__ double sum_of(const double *partial, unsigned count, double *waves) {
  double sum = 0.0;
  for (unsigned i = threadIdx.x; i < count; i += 256) sum += partial[i];
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  return (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

// The exponent e of the power of two that X0 is G times, and the factor that is left: 2^-e / (|G| + epsilon).
// (|G| 2^e is 128 to 256: far from what fp16 cannot hold at either end; and the factor at most 2^-7, so that its square, by which
// the first A is multiplied, is finite. Zeros have no such bound: they stay zeros by whatever they are multiplied, unless epsilon
// is zero too, and the formula says 0 / 0.)
__device__ __forceinline__ int exponent_and_factor(double sum, float epsilon, float *factor) {
  const double norm = __builtin_sqrt(sum);
  if (!(norm < __builtin_inf())) {   // an infinity or a NaN among the values: the result is NaN
    *factor = __builtin_nanf("");
    return 0;
  }
  if (norm == 0.0) {
    *factor = epsilon > 0.f ? 1.f : __builtin_nanf("");
    return 0;
  }
  int e = 0;
  (void)__builtin_frexp(norm, &e);
  e = 8 - e;
  *factor = (float)(__builtin_ldexp(1.0, -e) / (norm + (double)epsilon));
  return e;
}

// to[r][c] and to_t[c][r] = G[r][c] 2^e, 64 x 64 values a block, transposed through LDS. Bound by memory: 4096 x 8192 bf16
// 43 us, 4.7 TB/s.
template <int TYPE, bool PAIRS>
__global__ __launch_bounds__(256) void to_halves(const typename Value<TYPE>::type *in, size_t in_pitch, unsigned m, unsigned n,
                                                 _Float16 *to, unsigned to_pitch, size_t to_batch, size_t to_plane,
                                                 _Float16 *to_t, unsigned to_t_pitch, size_t to_t_batch, size_t to_t_plane,
                                                 const double *partial, unsigned count, float epsilon, float *factor) {
  using H = real::Halves<PAIRS>;
  using V = typename Value<TYPE>::type;
  typedef V eight_t __attribute__((ext_vector_type(8), aligned(sizeof(V))));
  __shared__ float tile[64][65];
  __shared__ double waves[4];
  const unsigned b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  float f;
  const int e = exponent_and_factor(sum_of(partial + (size_t)b * count, count, waves), epsilon, &f);
  if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) factor[b] = f;
  // (eight neighbours at a time; what is behind a row's end is written as the zero that it is)
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const unsigned r = q * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 8;
    const V *const from = in + ((size_t)b * m + r0 + r) * in_pitch + c0 + c;
    float v[8] = {};
    if (r0 + r < m) {
      if (c0 + c + 8 <= n) {
        const eight_t got = *reinterpret_cast<const eight_t *>(from);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_ldexpf((float)got[i], e);
      } else {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) {
          if (c0 + c + i < n) v[i] = __builtin_ldexpf((float)from[i], e);
        }
      }
      if (c0 + c < n) H::store(to + (size_t)b * to_batch + (size_t)(r0 + r) * to_pitch + c0 + c, to_plane, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) tile[r][c + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const unsigned r = (threadIdx.x & 7) * 8, c = q * 32 + (threadIdx.x >> 3);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[r + i][c];
    if (c0 + c < n && r0 + r < m) H::store(to_t + (size_t)b * to_t_batch + (size_t)(c0 + c) * to_t_pitch + r0 + r, to_t_plane, v);
  }
}

// ---- small matrices: all steps in one launch ----
// A workgroup of 16 waves has one matrix, whose chain stays in LDS: X and X^T, A and P, rows 16 bytes longer than a multiple of
// 64 bytes, so that the fragment reads of 16 rows fall on different banks. A wave computes 32 x 32 sums at a time; every
// product is at most two rounds of them. What bounds it is latency: 15 products one after the other, three barriers a step.
// 16 x 128 x 96 bf16: 80 us as 17 launches, 28 in one (64 x 480: 78 and 36).
constexpr unsigned kSmallWaves = 16, kSmallRounds = 2, kSmallPieces = 4, kSmallLds = 156 * 1024;
struct SmallSizes {
  unsigned mp, np;                 // extents padded to 32
  unsigned x_pitch, t_pitch;       // halves: rows of X (np + 8); rows of X^T, A and P (mp + 8)
  unsigned x_plane, t_plane, a_plane;
  unsigned bytes;
};
constexpr SmallSizes small_sizes(unsigned m, unsigned n, unsigned planes) {
  SmallSizes s = {};
  s.mp = (m + 31) / 32 * 32;
  s.np = (n + 31) / 32 * 32;
  s.x_pitch = s.np + 8;
  s.t_pitch = s.mp + 8;
  s.x_plane = s.mp * s.x_pitch;
  s.t_plane = s.np * s.t_pitch;
  s.a_plane = s.mp * s.t_pitch;
  s.bytes = planes * 2 * (s.x_plane + s.t_plane + 2 * s.a_plane) + 2 * s.mp * 4;
  return s;
}
bool fits_small(size_t m, size_t n, unsigned planes) {
  if (m > 256 || n > 4096) return false;
  const SmallSizes s = small_sizes((unsigned)m, (unsigned)n, planes);
  return s.bytes <= kSmallLds && (s.mp / 32) * (s.np / 32) <= kSmallWaves * kSmallRounds &&
         s.mp * s.np / 8 <= kSmallPieces * 64 * kSmallWaves;
}

struct SmallArgs {
  const void *in;
  void *out;
  size_t in_pitch, out_pitch;
  unsigned rows, cols;             // of the input
  int steps;
  float a, b, c, epsilon;
};

template <int TYPE>
__global__ __launch_bounds__(64 * kSmallWaves) void orthogonalize_small(SmallArgs args) {
  constexpr bool PAIRS = TYPE != kBfloat16;
  constexpr int PLANES = PAIRS ? 2 : 1;
  using H = real::Halves<PAIRS>;
  using V = typename Value<TYPE>::type;
  typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) char lds[kSmallLds];
  __shared__ double sums[kSmallWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  int fr = lane & 15, g = lane >> 4;
  const bool tall = args.rows > args.cols;
  const unsigned m = tall ? args.cols : args.rows, n = tall ? args.rows : args.cols;
  const SmallSizes z = small_sizes(m, n, PLANES);
  _Float16 *const x = reinterpret_cast<_Float16 *>(lds), *const t = x + PLANES * z.x_plane, *const a = t + PLANES * z.t_plane,
                  *const p = a + PLANES * z.a_plane;
  float *const diagonal = reinterpret_cast<float *>(p + PLANES * z.a_plane), *const diagonal_p = diagonal + z.mp;
  const V *const in = static_cast<const V *>(args.in) + (size_t)blockIdx.x * args.rows * args.in_pitch;

  // G, eight neighbours of a row at a time, neighbouring lanes in neighbouring rows (which spreads the transpose's writes over
  // the banks); read once
  typedef V eight_t __attribute__((ext_vector_type(8), aligned(sizeof(V))));
  const unsigned pieces = args.rows * ((args.cols + 7) / 8);
  float v[kSmallPieces][8];
  double sum = 0.0;
#pragma unroll
  for (unsigned q = 0; q < kSmallPieces; ++q) {
    const unsigned id = threadIdx.x + q * 64 * kSmallWaves;
    const unsigned c8 = id / args.rows, r = id - c8 * args.rows, c = c8 * 8;
    const V *const from = in + (size_t)r * args.in_pitch + c;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[q][e] = 0.f;
    if (id < pieces) {
      if (c + 8 <= args.cols) {
        const eight_t got = *reinterpret_cast<const eight_t *>(from);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = (float)got[e];
      } else {
#pragma unroll
        for (unsigned e = 0; e < 8; ++e) {
          if (c + e < args.cols) v[q][e] = (float)from[e];
        }
      }
    }
  }
  // zeros behind the ends of rows and columns
  for (unsigned i = threadIdx.x; i < z.bytes / 16; i += 64 * kSmallWaves) reinterpret_cast<int4_t *>(lds)[i] = int4_t{0, 0, 0, 0};
#pragma unroll
  for (unsigned q = 0; q < kSmallPieces; ++q) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)v[q][e], (double)v[q][e], sum);
  }
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0.0;
  for (unsigned w = 0; w < kSmallWaves; ++w) sum += sums[w];
  float factor;
  const int e2 = exponent_and_factor(sum, args.epsilon, &factor);
  {
    _Float16 *const same = tall ? t : x, *const turned = tall ? x : t;
    const unsigned same_pitch = tall ? z.t_pitch : z.x_pitch, turned_pitch = tall ? z.x_pitch : z.t_pitch;
    const unsigned same_plane = tall ? z.t_plane : z.x_plane, turned_plane = tall ? z.x_plane : z.t_plane;
#pragma unroll
    for (unsigned q = 0; q < kSmallPieces; ++q) {
      const unsigned id = threadIdx.x + q * 64 * kSmallWaves;
      const unsigned c8 = id / args.rows, r = id - c8 * args.rows, c = c8 * 8;
      if (id < pieces) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = __builtin_ldexpf(v[q][e], e2);
        H::store(same + r * same_pitch + c, same_plane, v[q]);       // (behind the row's end: zeros)
#pragma unroll
        for (int e = 0; e < 8; ++e) H::put(turned + (c + e) * turned_pitch + r, turned_plane, v[q][e]);
      }
    }
  }
  __syncthreads();

  // 32 x 32 sums D[y][x] of rows of `rx` (x) and of `ry` (y), over k: [16 of y][16 of x]
  auto multiply = [&](const _Float16 *rx, unsigned px, unsigned planex, const _Float16 *ry, unsigned py, unsigned planey, unsigned k,
                      real::float4_t (&d)[2][2]) __attribute__((always_inline)) {
    real::float4_t lo[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        d[j][i] = 0.f;
        lo[j][i] = 0.f;
      }
    }
    // (fragments are read one step of 32 ahead; behind the last one the last one's again)
    real::half8_t fx[PLANES][2], fy[PLANES][2], next_x[PLANES][2], next_y[PLANES][2];
    auto read = [&](unsigned at) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < PLANES; ++q) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          next_x[q][i] = *reinterpret_cast<const real::half8_t *>(rx + q * planex + (i * 16 + fr) * px + at + g * 8);
          next_y[q][i] = *reinterpret_cast<const real::half8_t *>(ry + q * planey + (i * 16 + fr) * py + at + g * 8);
        }
      }
    };
    read(0);
    for (unsigned at = 0; at < k; at += 32) {
#pragma unroll
      for (int q = 0; q < PLANES; ++q) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fx[q][i] = next_x[q][i];
          fy[q][i] = next_y[q][i];
        }
      }
      read(at + 32 < k ? at + 32 : at);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) d[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fx[0][i], fy[0][j], d[j][i], 0, 0, 0);
      }
      if constexpr (PAIRS) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            lo[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fx[0][i], fy[PLANES - 1][j], lo[j][i], 0, 0, 0);
            lo[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fx[PLANES - 1][i], fy[0][j], lo[j][i], 0, 0, 0);
          }
        }
      }
    }
    if constexpr (PAIRS) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) d[j][i] += lo[j][i] * 0x1p-11f;
      }
    }
  };
  auto load4 = [&](const _Float16 *from, unsigned plane, float (&v)[4]) {
    const half4_t h = *reinterpret_cast<const half4_t *>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)h[e];
    if constexpr (PAIRS) {
      const half4_t l = *reinterpret_cast<const half4_t *>(from + plane);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf((float)l[e], 0x1p-11f, v[e]);
    }
  };
  auto store4 = [&](_Float16 *to, unsigned plane, const float (&v)[4]) {
#pragma unroll
    for (int q = 0; q < PLANES; ++q) {
      const half4_t h = {H::part(v[0], q), H::part(v[1], q), H::part(v[2], q), H::part(v[3], q)};
      *reinterpret_cast<half4_t *>(to + q * plane) = h;
    }
  };

  const unsigned bm = z.mp / 32, bn = z.np / 32;
  float f = factor;
  real::float4_t d[kSmallRounds][2][2];
  // X's new values of piece (i, j) of a round
  auto updated = [&](unsigned round, unsigned block, int j, int i, float (&w)[4]) __attribute__((always_inline)) {
    const unsigned y = block / bn * 32 + j * 16 + fr, c = block % bn * 32 + i * 16 + g * 4;
    const float dy = args.a + diagonal_p[y];
    float old[4];
    load4(x + y * z.x_pitch + c, z.x_plane, old);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = f * __builtin_fmaf(dy, old[e], d[round][j][i][e]);
  };
#pragma unroll 1
  for (int step = 0;;) {
    // (addresses are worked out anew in every step: kept through the loop they fill the registers)
    asm volatile("" : "+v"(fr), "+v"(g));
    // A: its diagonal apart (all of it: the mirrored half costs no round more)
#pragma unroll 1
    for (unsigned block = wave; block < bm * bm; block += kSmallWaves) {
      const unsigned y0 = block / bm * 32, x0 = block % bm * 32;
      real::float4_t v[2][2];
      multiply(x + x0 * z.x_pitch, z.x_pitch, z.x_plane, x + y0 * z.x_pitch, z.x_pitch, z.x_plane, z.np, v);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned y = y0 + j * 16 + fr, c = x0 + i * 16 + g * 4;
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = f * f * v[j][i][e];
            if (c + e == y) {
              diagonal[y] = w[e];
              w[e] = 0.f;
            }
          }
          store4(a + y * z.t_pitch + c, z.a_plane, w);
        }
      }
    }
    __syncthreads();
    // P
#pragma unroll 1
    for (unsigned block = wave; block < bm * bm; block += kSmallWaves) {
      const unsigned y0 = block / bm * 32, x0 = block % bm * 32;
      real::float4_t v[2][2];
      multiply(a + x0 * z.t_pitch, z.t_pitch, z.a_plane, a + y0 * z.t_pitch, z.t_pitch, z.a_plane, z.mp, v);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const unsigned y = y0 + j * 16 + fr;
        const float dy = diagonal[y];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned c = x0 + i * 16 + g * 4;
          float old[4], w[4];
          load4(a + y * z.t_pitch + c, z.a_plane, old);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = __builtin_fmaf(args.c, __builtin_fmaf(dy + diagonal[c + e], old[e], v[j][i][e]), args.b * old[e]);
            if (c + e == y) {
              diagonal_p[y] = __builtin_fmaf(args.c, __builtin_fmaf(dy, dy, v[j][i][e]), args.b * dy);
              w[e] = 0.f;
            }
          }
          store4(p + y * z.t_pitch + c, z.a_plane, w);
        }
      }
    }
    __syncthreads();
    // X and X^T, which are written only when everybody has read them
#pragma unroll
    for (unsigned round = 0; round < kSmallRounds; ++round) {
      const unsigned block = wave + round * kSmallWaves;
      if (block < bm * bn) {
        const unsigned y0 = block / bn * 32, x0 = block % bn * 32;
        multiply(t + x0 * z.t_pitch, z.t_pitch, z.t_plane, p + y0 * z.t_pitch, z.t_pitch, z.a_plane, z.mp, d[round]);
      }
    }
    if (++step == args.steps) break;
    __syncthreads();
#pragma unroll
    for (unsigned round = 0; round < kSmallRounds; ++round) {
      const unsigned block = wave + round * kSmallWaves;
      if (block < bm * bn) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned y = block / bn * 32 + j * 16 + fr, c = block % bn * 32 + i * 16 + g * 4;
            float w[4];
            updated(round, block, j, i, w);
            store4(x + y * z.x_pitch + c, z.x_plane, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) H::put(t + (c + e) * z.t_pitch + y, z.t_plane, w[e]);
          }
        }
      }
    }
    f = 1.f;
    __syncthreads();
  }
  V *const out = static_cast<V *>(args.out) + (size_t)blockIdx.x * args.rows * args.out_pitch;
#pragma unroll
  for (unsigned round = 0; round < kSmallRounds; ++round) {
    const unsigned block = wave + round * kSmallWaves;
    if (block < bm * bn) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned y = block / bn * 32 + j * 16 + fr, c = block % bn * 32 + i * 16 + g * 4;
          float w[4];
          updated(round, block, j, i, w);
          if (y >= m || c >= n) continue;
          if (tall) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (c + e < n) out[(size_t)(c + e) * args.out_pitch + y] = (V)w[e];
            }
          } else {
            real::store_row(out + (size_t)y * args.out_pitch + c, n - c, w);
          }
        }
      }
    }
  }
}

// Where things are in the workspace.
struct Layout {
  size_t m, n;                             // shorter and longer extent
  bool tall;                               // the input has more rows than columns
  int planes;
  size_t mp, np;                           // pitches, elements
  size_t x_plane, t_plane, a_plane;        // elements of one plane of one matrix
  size_t counters, partial, norm, factor, diagonal, x, t0, t1, a, p, bytes;
  size_t zeroed;
  unsigned norm_x, norm_y, norm_rows;      // partial sums of squares, rows of one
};

struct Product {
  RealGemmPlan plan;
  unsigned blocks_x, blocks_y;
  size_t blocks;                           // in all
};

// (the shapes of orthogonalize.h, in their order; the figures are estimates from a trace of a few sizes, see real_plan.h)
constexpr RealShape kHalfShapes[] = {{256, 256, 512, 1, 1.0f, 1.55f, 14.0f, 0.8f, "256x256"},
                                     {128, 128, 256, 2, 0.62f, 0.87f, 9.0f, 1.3f, "128x128"},
                                     {64, 64, 256, 2, 0.18f, 0.27f, 5.0f, 2.6f, "64x64"},
                                     {128, 128, 512, 1, 0.35f, 0.54f, 7.0f, 1.3f, "128x128 8-wave"},
                                     {192, 192, 512, 1, 0.62f, 0.97f, 11.0f, 1.0f, "192x192"}};
constexpr RealShape kPairsShapes[] = {{128, 128, 512, 1, 1.15f, 1.40f, 7.0f, 1.3f, "128x128"},
                                      {64, 64, 256, 2, 0.50f, 0.80f, 6.0f, 2.6f, "64x64"}};
#define CCGLIB_SAME(ID, BX, BY, WX, WY, SLOTS, EU) \
  static_assert(CCGLIB_TABLE[ID].bx == BX && CCGLIB_TABLE[ID].by == BY && CCGLIB_TABLE[ID].threads == 64 * WX * WY, \
                "the table is in the order of the shapes");
#define CCGLIB_TABLE kHalfShapes
CCGLIB_HALF_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#define CCGLIB_TABLE kPairsShapes
CCGLIB_HALF_PAIRS_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#undef CCGLIB_SAME

Product plan_product(const OrthogonalizeParams &p, size_t nx, size_t ny, size_t k, bool symmetric) {
  const bool pairs = as_pairs(p.type);
  const size_t batch = p.batch;
  const RealShape *const shapes = pairs ? kPairsShapes : kHalfShapes;
  const int count = pairs ? (int)(sizeof kPairsShapes / sizeof kPairsShapes[0]) : (int)(sizeof kHalfShapes / sizeof kHalfShapes[0]);
  Product r = {};
  r.plan = plan_real_gemm(shapes, count, batch, nx, ny, ceil_div(k, (size_t)64), symmetric, p.block_option);
  const RealShape &s = shapes[r.plan.shape];
  r.blocks_x = (unsigned)ceil_div(nx, s.bx);
  r.blocks_y = (unsigned)ceil_div(ny, s.by);
  r.blocks = real_blocks(s, batch, nx, ny, symmetric);
  return r;
}

Layout layout_of(const OrthogonalizeParams &p) {
  Layout l = {};
  l.tall = p.m > p.n;
  l.m = std::min(p.m, p.n);
  l.n = std::max(p.m, p.n);
  const bool pairs = as_pairs(p.type);
  l.planes = pairs ? 2 : 1;
  l.mp = up(l.m, 64);
  l.np = up(l.n, 64);
  l.x_plane = l.m * l.np;
  l.t_plane = l.n * l.mp;
  l.a_plane = l.m * l.mp;
  l.norm_x = (unsigned)ceil_div(p.n, (size_t)kNormColumns);
  // (at least 8 rows, and at most about 1024 partial sums, which every block of to_halves adds up)
  l.norm_rows = (unsigned)std::max<size_t>(8, ceil_div((size_t)p.m * l.norm_x, 1024));
  l.norm_y = (unsigned)ceil_div(p.m, (size_t)l.norm_rows);
  size_t counters = 0, partial = 0;
  const Product products[] = {plan_product(p, l.m, l.m, l.n, true), plan_product(p, l.m, l.m, l.m, true),
                              plan_product(p, l.n, l.m, l.m, false),
                              plan_product(p, l.m, l.n, l.m, false)};
  for (const Product &r : products) {
    counters = std::max(counters, r.plan.counter_bytes);
    partial = std::max(partial, r.plan.partial_bytes);
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += up(bytes, kAlign);
    return here;
  };
  const size_t h = sizeof(_Float16) * l.planes * p.batch;
  l.counters = take(counters);
  // (the ends of rows, up to a whole 16 bytes of K, are read and hold zeros; so do those of diagonals)
  l.x = take(l.x_plane * h);
  l.t0 = take(l.t_plane * h);
  l.t1 = take(l.t_plane * h);
  l.a = take(l.a_plane * h);
  l.p = take(l.a_plane * h);
  l.diagonal = take(2 * p.batch * l.mp * sizeof(float));
  l.zeroed = at;
  l.partial = take(partial);
  l.norm = take((size_t)p.batch * l.norm_x * l.norm_y * sizeof(double));
  l.factor = take(p.batch * sizeof(float));
  l.bytes = at;
  return l;
}

bool is_small(const OrthogonalizeParams &p) {
  return !p.block_option && fits_small(std::min(p.m, p.n), std::max(p.m, p.n), as_pairs(p.type) ? 2 : 1);
}

// Whether the one launch may not be used in place: its workgroups read and write a matrix each on their own, and a matrix of the
// output then lies on another one of the input. (Several launches have read all of the input before the first writes.)
bool meets_another_in_place(const OrthogonalizeParams &p) { return p.batch > 1 && p.in_pitch != p.out_pitch; }

template <bool PAIRS, int STEP>
hipError_t launch_product(const Product &r, const real::Args &a, const typename real::StoreChain<PAIRS, STEP>::Params &e,
                          hipStream_t stream) {
  using Store = real::StoreChain<PAIRS, STEP>;
  const unsigned grid = (unsigned)(r.blocks * r.plan.parts);
  if constexpr (PAIRS) {
    switch (r.plan.shape) {
#define CCGLIB_CASE(ID, BX, BY, WX, WY, SLOTS, EU)                                                                        \
  case ID:                                                                                                                \
    real::gemm_real<real::kHalfPairs, 0, 0, BX, BY, WX, WY, SLOTS, EU, Store><<<grid, 64 * WX * WY, 0, stream>>>(a, e); \
    break;
      CCGLIB_HALF_PAIRS_SHAPES(CCGLIB_CASE)
#undef CCGLIB_CASE
    }
  } else {
    switch (r.plan.shape) {
#define CCGLIB_CASE(ID, BX, BY, WX, WY, SLOTS, EU)                                                                   \
  case ID:                                                                                                           \
    real::gemm_real<real::kHalf, 0, 0, BX, BY, WX, WY, SLOTS, EU, Store><<<grid, 64 * WX * WY, 0, stream>>>(a, e); \
    break;
      CCGLIB_HALF_SHAPES(CCGLIB_CASE)
#undef CCGLIB_CASE
    }
  }
  return hipGetLastError();
}

template <int TYPE> hipError_t launch(const OrthogonalizeParams &p, hipStream_t stream) {
  constexpr bool PAIRS = TYPE != kBfloat16;
  using V = typename Value<TYPE>::type;
  if (is_small(p) && !(p.in == p.out && meets_another_in_place(p))) {
    SmallArgs a = {p.in, p.out, p.in_pitch, p.out_pitch, p.m, p.n, p.steps, p.a, p.b, p.c, p.epsilon};
    orthogonalize_small<TYPE><<<p.batch, 64 * kSmallWaves, 0, stream>>>(a);
    return hipGetLastError();
  }
  const Layout l = layout_of(p);
  char *const ws = static_cast<char *>(p.workspace);
  auto halves = [&](size_t at) { return reinterpret_cast<_Float16 *>(ws + at); };
  double *const norm = reinterpret_cast<double *>(ws + l.norm);
  float *const factor = reinterpret_cast<float *>(ws + l.factor), *const diagonal = reinterpret_cast<float *>(ws + l.diagonal);
  _Float16 *const x = halves(l.x), *const a = halves(l.a), *const pp = halves(l.p);
  _Float16 *t = halves(l.t0), *t_next = halves(l.t1);
  const V *in = static_cast<const V *>(p.in);
  const size_t pl = PAIRS ? 2 : 1;
  const size_t xb = l.x_plane * pl, tb = l.t_plane * pl, ab = l.a_plane * pl;

  sum_of_squares<TYPE><<<dim3(l.norm_x, l.norm_y, p.batch), 256, 0, stream>>>(in, p.in_pitch, p.m, p.n, l.norm_rows, norm);
  const dim3 tiles((unsigned)ceil_div(p.n, (size_t)64), (unsigned)ceil_div(p.m, (size_t)64), p.batch);
  if (l.tall) {
    to_halves<TYPE, PAIRS><<<tiles, 256, 0, stream>>>(in, p.in_pitch, p.m, p.n, t, l.mp, tb, l.t_plane, x, l.np, xb, l.x_plane,
                                                      norm, l.norm_x * l.norm_y, p.epsilon, factor);
  } else {
    to_halves<TYPE, PAIRS><<<tiles, 256, 0, stream>>>(in, p.in_pitch, p.m, p.n, x, l.np, xb, l.x_plane, t, l.mp, tb, l.t_plane,
                                                      norm, l.norm_x * l.norm_y, p.epsilon, factor);
  }
  HIP_PASS(hipGetLastError());

  struct Matrix {
    const _Float16 *at;
    size_t rows, pitch, plane, batch;
  };
  const Product gram = plan_product(p, l.m, l.m, l.n, true), square = plan_product(p, l.m, l.m, l.m, true);
  const Product update = plan_product(p, l.n, l.m, l.m, false), narrow = plan_product(p, l.m, l.n, l.m, false);
  auto args = [&](const Matrix &mx, const Matrix &my, size_t k, const Product &r, bool symmetric) {
    real::Args g = {};
    g.x = reinterpret_cast<const char *>(mx.at);
    g.y = reinterpret_cast<const char *>(my.at);
    g.nx = (unsigned)mx.rows;
    g.ny = (unsigned)my.rows;
    g.batch = p.batch;
    g.x_pitch = (unsigned)mx.pitch * 2;
    g.y_pitch = (unsigned)my.pitch * 2;
    g.x_batch = mx.batch * 2;
    g.y_batch = my.batch * 2;
    g.x_plane = mx.plane * 2;
    g.y_plane = my.plane * 2;
    g.k_bytes = (unsigned)up(k, 64) * 2;   // (rows are padded to whole pieces, with zeros)
    g.pieces = (unsigned)ceil_div(g.k_bytes, (size_t)real::kPieceBytes);
    g.blocks_x = r.blocks_x;
    g.blocks_y = r.blocks_y;
    g.symmetric = symmetric;
    g.parts = r.plan.parts;
    g.pieces_per_part = r.plan.pieces_per_part;
    g.arrived = reinterpret_cast<unsigned *>(ws + l.counters);
    g.partial = reinterpret_cast<float *>(ws + l.partial);
    return g;
  };
  for (int step = 0; step < p.steps; ++step) {
    const bool first = step == 0, last = step + 1 == p.steps;
    const Matrix mx{x, l.m, l.np, l.x_plane, xb}, mt{t, l.n, l.mp, l.t_plane, tb}, ma{a, l.m, l.mp, l.a_plane, ab},
        mp{pp, l.m, l.mp, l.a_plane, ab};
    auto fill = [&](auto &e, const Matrix *to, _Float16 *at, const Matrix *o, size_t nx, size_t ny) {
      e.a = p.a;
      e.b = p.b;
      e.c = p.c;
      e.nx = (unsigned)nx;
      e.ny = (unsigned)ny;
      e.diagonal = diagonal;
      e.diagonal_p = diagonal + (size_t)p.batch * l.mp;
      e.diagonal_pitch = (unsigned)l.mp;
      if (to) {
        e.to = at;
        e.to_pitch = (unsigned)to->pitch;
        e.to_plane = to->plane;
        e.to_batch = to->batch;
      }
      if (o) {
        e.old = o->at;
        e.old_pitch = (unsigned)o->pitch;
        e.old_plane = o->plane;
        e.old_batch = o->batch;
      }
    };
    typename real::StoreChain<PAIRS, real::kGram>::Params eg = {};
    fill(eg, &ma, a, nullptr, l.m, l.m);
    eg.factor = first ? factor : nullptr;
    HIP_PASS((launch_product<PAIRS, real::kGram>(gram, args(mx, mx, l.n, gram, true), eg, stream)));
    typename real::StoreChain<PAIRS, real::kSquare>::Params es = {};
    fill(es, &mp, pp, &ma, l.m, l.m);
    HIP_PASS((launch_product<PAIRS, real::kSquare>(square, args(ma, ma, l.m, square, true), es, stream)));
    if (last && l.tall) {   // (rows of X^T P: the caller's orientation)
      typename real::StoreChain<PAIRS, real::kUpdateT>::Params e = {};
      fill(e, nullptr, nullptr, &mt, l.m, l.n);
      e.factor = first ? factor : nullptr;
      e.out = p.out;
      e.out_pitch = p.out_pitch;
      e.out_batch = (size_t)p.m * p.out_pitch;
      e.out_type = p.type;
      return launch_product<PAIRS, real::kUpdateT>(narrow, args(mp, mt, l.m, narrow, false), e, stream);
    }
    typename real::StoreChain<PAIRS, real::kUpdate>::Params e = {};
    fill(e, &mx, x, &mx, l.n, l.m);   // (each value is read, then written, by the same lane)
    e.factor = first ? factor : nullptr;
    if (last) {
      e.out = p.out;
      e.out_pitch = p.out_pitch;
      e.out_batch = (size_t)p.m * p.out_pitch;
      e.out_type = p.type;
    }
    e.to_t = t_next;
    e.to_t_pitch = (unsigned)l.mp;
    e.to_t_plane = l.t_plane;
    e.to_t_batch = tb;
    HIP_PASS((launch_product<PAIRS, real::kUpdate>(update, args(mt, mp, l.m, update, false), e, stream)));
    std::swap(t, t_next);
  }
  return hipSuccess;
}

}  // namespace

size_t orthogonalize_workspace_bytes(const OrthogonalizeParams &p) {
  return is_small(p) && !meets_another_in_place(p) ? 0 : layout_of(p).bytes;
}
size_t orthogonalize_zeroed_bytes(const OrthogonalizeParams &p) {
  return is_small(p) && !meets_another_in_place(p) ? 0 : layout_of(p).zeroed;
}

hipError_t launch_orthogonalize(const OrthogonalizeParams &p, hipStream_t stream) {
  if (p.batch == 0 || p.m == 0 || p.n == 0) return hipSuccess;
  switch (p.type) {
    case kFloat32: return launch<kFloat32>(p, stream);
    case kFloat16: return launch<kFloat16>(p, stream);
    default: return launch<kBfloat16>(p, stream);
  }
}

}  // namespace ccglib_amd
