// Combine: out[t] = sum over j of w[t][j] y[slot[t][j]], and the way back: dy[slot] = w dout[t], dw[t][j] = <dout[t], y[slot]>.
// Sums are 32 bits, in the order of j. A slot that is no row of y counts as a row of zeros.
//
// Bound by memory: a row of y is read once and used once. 64 or 256 threads have a token (up to 512 columns, and from there on), 8 neighbouring columns a
// thread at a time, and all its rows' loads are on their way together. 4099 tokens, 2 rows of 4104 each: 17.0 us, 5.9 TB/s (part of y
// is still in the last-level cache); the way back of 16384 tokens, 4 rows of 4096 each, with dw: 241 us, 5.0 TB/s.
#include "linear_gemm.h"
#include "route.h"

namespace ccglib_amd {
namespace {

using linear::Value;

struct CombineArgs {
  const char *y, *dout;
  const int *slots;
  const float *weights;          // null: 1
  char *out;                     // of the sums; of the way back: dy
  float *dweights;
  unsigned tokens, k, n, rows;
  size_t y_pitch, out_pitch;
};

// The token's rows, in registers that are the same for all threads of it.
template <int K> struct Rows {
  unsigned slot[K];
  float w[K];
  __device__ __forceinline__ Rows(const CombineArgs &a, unsigned t) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      slot[j] = (unsigned)j < a.k ? (unsigned)a.slots[(size_t)t * a.k + j] : 0xffffffffu;
      w[j] = (unsigned)j < a.k && a.weights ? a.weights[(size_t)t * a.k + j] : 1.f;
    }
  }
};

template <int TYPE, int K, int THREADS> __global__ __launch_bounds__(256) void combine_sums(CombineArgs a) {
  using T = typename Value<TYPE>::type;
  const unsigned t = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (t >= a.tokens) return;
  const Rows<K> r(a, t);
  for (unsigned x = threadIdx.x % THREADS * 8; x < a.n; x += THREADS * 8) {
    float s[8] = {}, v[K][8];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (r.slot[j] < a.rows) linear::load_row(reinterpret_cast<const T *>(a.y) + (size_t)r.slot[j] * a.y_pitch + x, a.n - x, v[j]);
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (r.slot[j] < a.rows) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = __builtin_fmaf(r.w[j], v[j][e], s[e]);
      }
    }
    real::store_row(reinterpret_cast<T *>(a.out) + (size_t)t * a.out_pitch + x, a.n - x, s);
  }
}

template <int TYPE, int K, int THREADS> __global__ __launch_bounds__(256) void combine_backward(CombineArgs a) {
  using T = typename Value<TYPE>::type;
  const unsigned t = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (THREADS == 64 && t >= a.tokens) return;      // (256: a block has one token)
  const Rows<K> r(a, t);
  float dots[K] = {};
  for (unsigned x = threadIdx.x % THREADS * 8; x < a.n; x += THREADS * 8) {
    float d[8], v[K][8];
    linear::load_row(reinterpret_cast<const T *>(a.dout) + (size_t)t * a.out_pitch + x, a.n - x, d);
    if (a.y) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (r.slot[j] < a.rows) linear::load_row(reinterpret_cast<const T *>(a.y) + (size_t)r.slot[j] * a.y_pitch + x, a.n - x, v[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (r.slot[j] >= a.rows) continue;
      if (a.y) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dots[j] = __builtin_fmaf(v[j][e], d[e], dots[j]);
      }
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = r.w[j] * d[e];
      if (a.out) real::store_row(reinterpret_cast<T *>(a.out) + (size_t)r.slot[j] * a.y_pitch + x, a.n - x, w);
    }
  }
  if (!a.dweights) return;
#pragma unroll
  for (int j = 0; j < K; ++j) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) dots[j] += __shfl_xor(dots[j], d);
  }
  const unsigned lane = threadIdx.x & 63;
  if constexpr (THREADS == 256) {
    __shared__ float waves[4][K];
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < K; ++j) waves[threadIdx.x >> 6][j] = dots[j];
    }
    __syncthreads();
    if (threadIdx.x < a.k) {
      const unsigned j = threadIdx.x;
      a.dweights[(size_t)t * a.k + j] = (waves[0][j] + waves[1][j]) + (waves[2][j] + waves[3][j]);
    }
  } else {
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if ((unsigned)j < a.k) a.dweights[(size_t)t * a.k + j] = dots[j];
      }
    }
  }
}

// Calls `f` with the type, the rows of a token (the next power of two) and its threads.
template <typename F> void by_sizes(const CombineParams &p, F &&f) {
  using std::integral_constant;
  auto threads = [&](auto type, auto k) {
    if (p.n <= 512) return f(type, k, integral_constant<int, 64>{});
    return f(type, k, integral_constant<int, 256>{});
  };
  auto chosen = [&](auto type) {
    if (p.chosen <= 1) return threads(type, integral_constant<int, 1>{});
    if (p.chosen <= 2) return threads(type, integral_constant<int, 2>{});
    if (p.chosen <= 4) return threads(type, integral_constant<int, 4>{});
    if (p.chosen <= 8) return threads(type, integral_constant<int, 8>{});
    return threads(type, integral_constant<int, 16>{});
  };
  if (p.type == kFloat16) return chosen(integral_constant<int, kFloat16>{});
  return chosen(integral_constant<int, kBfloat16>{});
}

CombineArgs args_of(const CombineParams &p, const int *slots, const float *weights) {
  CombineArgs a = {};
  a.slots = slots;
  a.weights = weights;
  a.tokens = p.tokens;
  a.k = p.chosen;
  a.n = p.n;
  a.rows = p.rows;
  a.y_pitch = p.y_pitch;
  a.out_pitch = p.out_pitch;
  return a;
}

}  // namespace

hipError_t launch_combine(const CombineParams &p, const void *y, const int *slots, const float *weights, void *out, hipStream_t stream) {
  if (p.tokens == 0 || p.n == 0) return hipSuccess;
  CombineArgs a = args_of(p, slots, weights);
  a.y = static_cast<const char *>(y);
  a.out = static_cast<char *>(out);
  by_sizes(p, [&](auto type, auto k, auto threads) {
    constexpr int THREADS = decltype(threads)::value;
    combine_sums<decltype(type)::value, decltype(k)::value, THREADS>
        <<<(unsigned)ceil_div(p.tokens, (size_t)(256 / THREADS)), 256, 0, stream>>>(a);
  });
  return hipGetLastError();
}

hipError_t launch_combine_backward(const CombineParams &p, const void *dout, const void *y, const int *slots, const float *weights,
                                   void *dy, float *dweights, hipStream_t stream) {
  if (p.tokens == 0) return hipSuccess;
  CombineArgs a = args_of(p, slots, weights);
  a.dout = static_cast<const char *>(dout);
  a.y = static_cast<const char *>(y);
  a.out = static_cast<char *>(dy);
  a.dweights = dweights;
  by_sizes(p, [&](auto type, auto k, auto threads) {
    constexpr int THREADS = decltype(threads)::value;
    combine_backward<decltype(type)::value, decltype(k)::value, THREADS>
        <<<(unsigned)ceil_div(p.tokens, (size_t)(256 / THREADS)), 256, 0, stream>>>(a);
  });
  return hipGetLastError();
}

}  // namespace ccglib_amd
