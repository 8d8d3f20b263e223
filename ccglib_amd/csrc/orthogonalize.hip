// Orthogonalised updates: X0 = G / (|G| + epsilon) (G^T where that is the wider one), |.| the Frobenius norm, then steps of
//   A = X X^T,  P = b A + c A A,  X <- a X + P X,
// which drive every singular value of X towards 1 (a Newton-Schulz iteration of degree five).
//
// All three products run on gemm_real. A and P are symmetric: blocks below the diagonal are multiplied, and stored twice;
// their diagonals are kept apart, in 32 bits.
// P X needs X with its columns contiguous, so X is kept in both orientations, and the epilogue of P X writes both.
//
// bf16 updates: the chain is fp16 (11 bits where the update has 8), sums are 32 bits. X0 is G times a power of two, which
// loses nothing; the rest of 1 / (|G| + epsilon) is a factor of the first step's epilogues. fp16 and fp32 updates: every
// value of the chain is two fp16, 22 bits, and three of the four products are added up (the fourth is 2^-22 of the first).
// |G| is summed in 64 bits, so that no G overflows it.
#include <algorithm>

#include "orthogonalize.h"
#include "real_plan.h"

namespace ccglib_amd {
namespace {

constexpr size_t kAlign = 256;
size_t up(size_t n, size_t to) { return ceil_div(n, to) * to; }

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
// neighbours at a time
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
// (|G| 2^e is 128 to 256: far from what fp16 cannot hold at either end)
__device__ __forceinline__ int exponent_and_factor(double sum, float epsilon, float *factor) {
  const double norm = __builtin_sqrt(sum);
  if (!(norm < __builtin_inf())) {   // an infinity or a NaN among the values: the result is NaN
    *factor = __builtin_nanf("");
    return 0;
  }
  int e = 0;
  if (norm > 0.0) (void)__builtin_frexp(norm, &e);
  e = 8 - e;
  *factor = (float)(__builtin_ldexp(1.0, -e) / (norm + (double)epsilon));
  return e;
}

// to[r][c] and to_t[c][r] = G[r][c] 2^e, 64 x 64 values a block
template <int TYPE, bool PAIRS>
__global__ __launch_bounds__(256) void to_halves(const typename Value<TYPE>::type *in, size_t in_pitch, unsigned m, unsigned n,
                                                 _Float16 *to, unsigned to_pitch, size_t to_batch, size_t to_plane,
                                                 _Float16 *to_t, unsigned to_t_pitch, size_t to_t_batch, size_t to_t_plane,
                                                 const double *partial, unsigned count, float epsilon, float *factor) {
  using H = real::Halves<PAIRS>;
  __shared__ float tile[64][65];
  __shared__ double waves[4];
  const unsigned b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  float f;
  const int e = exponent_and_factor(sum_of(partial + (size_t)b * count, count, waves), epsilon, &f);
  if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) factor[b] = f;
  const int c = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < 64; r += 4) {
    if (r0 + r < m && c0 + c < n) {
      const float v = __builtin_ldexpf((float)in[((size_t)b * m + r0 + r) * in_pitch + c0 + c], e);
      tile[r][c] = v;
      H::put(to + (size_t)b * to_batch + (size_t)(r0 + r) * to_pitch + c0 + c, to_plane, v);
    }
  }
  __syncthreads();
  for (int r = threadIdx.x >> 6; r < 64; r += 4) {
    if (c0 + r < n && r0 + c < m) {
      H::put(to_t + (size_t)b * to_t_batch + (size_t)(c0 + r) * to_t_pitch + r0 + c, to_t_plane, tile[c][r]);
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

// (the shapes of orthogonalize.h, in their order; see real_plan.h for the figures)
constexpr RealShape kHalfShapes[] = {{256, 256, 1, 1.0f, 1.55f, 14.0f, 0.8f, "256x256"},
                                     {128, 128, 2, 0.62f, 0.87f, 9.0f, 1.3f, "128x128"},
                                     {64, 64, 2, 0.18f, 0.30f, 5.0f, 2.6f, "64x64"}};
constexpr RealShape kPairsShapes[] = {{128, 128, 1, 1.15f, 1.40f, 7.0f, 1.3f, "128x128"},
                                      {64, 64, 2, 0.50f, 0.80f, 6.0f, 2.6f, "64x64"}};
#define CCGLIB_SAME(ID, BX, BY, WX, WY, SLOTS, EU) \
  static_assert(CCGLIB_TABLE[ID].bx == BX && CCGLIB_TABLE[ID].by == BY, "the table is in the order of the shapes");
#define CCGLIB_TABLE kHalfShapes
CCGLIB_HALF_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#define CCGLIB_TABLE kPairsShapes
CCGLIB_HALF_PAIRS_SHAPES(CCGLIB_SAME)
#undef CCGLIB_TABLE
#undef CCGLIB_SAME

Product plan_product(bool pairs, size_t batch, size_t nx, size_t ny, size_t k, bool symmetric) {
  const RealShape *const shapes = pairs ? kPairsShapes : kHalfShapes;
  const int count = pairs ? (int)(sizeof kPairsShapes / sizeof kPairsShapes[0]) : (int)(sizeof kHalfShapes / sizeof kHalfShapes[0]);
  Product r = {};
  r.plan = plan_real_gemm(shapes, count, batch, nx, ny, ceil_div(k, (size_t)64), symmetric);
  const RealShape &s = shapes[r.plan.shape];
  r.blocks_x = (unsigned)ceil_div(nx, s.bx);
  r.blocks_y = (unsigned)ceil_div(ny, s.by);
  r.blocks = real_blocks(s, batch, nx, ny, symmetric);
  return r;
}

bool as_pairs(int type) { return type != kBfloat16; }

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
  // (at least 16 rows, and at most about 2048 partial sums, which every block of to_halves adds up)
  l.norm_rows = (unsigned)std::max<size_t>(16, ceil_div((size_t)p.m * l.norm_x, 2048));
  l.norm_y = (unsigned)ceil_div(p.m, (size_t)l.norm_rows);
  size_t counters = 0, partial = 0;
  const Product products[] = {plan_product(pairs, p.batch, l.m, l.m, l.n, true), plan_product(pairs, p.batch, l.m, l.m, l.m, true),
                              plan_product(pairs, p.batch, l.n, l.m, l.m, false),
                              plan_product(pairs, p.batch, l.m, l.n, l.m, false)};
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
  const Product gram = plan_product(PAIRS, p.batch, l.m, l.m, l.n, true), square = plan_product(PAIRS, p.batch, l.m, l.m, l.m, true);
  const Product update = plan_product(PAIRS, p.batch, l.n, l.m, l.m, false), narrow = plan_product(PAIRS, p.batch, l.m, l.n, l.m, false);
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

size_t orthogonalize_workspace_bytes(const OrthogonalizeParams &p) { return layout_of(p).bytes; }
size_t orthogonalize_zeroed_bytes(const OrthogonalizeParams &p) { return layout_of(p).zeroed; }

hipError_t launch_orthogonalize(const OrthogonalizeParams &p, hipStream_t stream) {
  if (p.batch == 0 || p.m == 0 || p.n == 0) return hipSuccess;
  switch (p.type) {
    case kFloat32: return launch<kFloat32>(p, stream);
    case kFloat16: return launch<kFloat16>(p, stream);
    default: return launch<kBfloat16>(p, stream);
  }
}

}  // namespace ccglib_amd
