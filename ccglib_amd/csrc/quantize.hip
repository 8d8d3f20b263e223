// Conversion to 8 bits with a scale for each group of 128 values of a row, or of 128 x 128 values; of a matrix, of its
// transpose, or of both in one pass over it. With t the largest value of the type:
//   amax = max(2^-100, largest finite |x| of the group)
//   float32 scales:  scale = amax / t, factor = t / amax   (each rounded once, to 32 bits)
//   e8m0 scales:     scale = 2^ceil(log2(amax / t)), factor = 1 / scale
//   q = 8-bit value nearest to x * factor, ties to even; NaN stays NaN, infinity stays infinity or, in e4m3, is NaN
// Values that are not finite leave the scale of their group alone. The bound is memory: 2 bytes in and 1 or 2 out a value.
#include <type_traits>

#include "scaled.h"

namespace ccglib_amd {
namespace {

typedef unsigned uint2_t __attribute__((ext_vector_type(2)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
typedef unsigned uint4_unaligned_t __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kGroup = (int)kScaleGroup;
constexpr float kSmallest = 0x1p-100f;

struct Args {
  const char *in;
  unsigned char *out, *out_t;
  char *scales, *scales_t;
  unsigned batch, m, n;
  size_t in_pitch;
  unsigned out_pitch, out_t_pitch, scales_pitch, scales_t_pitch;
  unsigned tiles_m, tiles_n;
};

template <int TYPE> struct Loaded;
template <> struct Loaded<kFloat32> { using type = float; };
template <> struct Loaded<kFloat16> { using type = _Float16; };
template <> struct Loaded<kBfloat16> { using type = __bf16; };

// Eight values from p on, of which `valid` are there; the others are zero.
template <int TYPE>
__device__ __forceinline__ void load8(const typename Loaded<TYPE>::type *p, int valid, float (&v)[8]) {
  if (valid >= 8) {
    if constexpr (TYPE == kFloat32) {
      const uint4_unaligned_t a = reinterpret_cast<const uint4_unaligned_t *>(p)[0];
      const uint4_unaligned_t b = reinterpret_cast<const uint4_unaligned_t *>(p)[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned lo = a[e], hi = b[e];
        v[e] = __builtin_bit_cast(float, lo);
        v[4 + e] = __builtin_bit_cast(float, hi);
      }
    } else {
      const uint4_unaligned_t a = *reinterpret_cast<const uint4_unaligned_t *>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned w = a[e];
        if constexpr (TYPE == kBfloat16) {
          v[2 * e] = __builtin_bit_cast(float, w << 16);
          v[2 * e + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
        } else {
          v[2 * e] = (float)__builtin_bit_cast(_Float16, (unsigned short)w);
          v[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < valid ? (float)p[e] : 0.f;
  }
}

__device__ __forceinline__ float finite_magnitude(float x) {
  const float m = __builtin_fabsf(x);
  return m < __builtin_inff() ? m : 0.f;
}

// Maximum over each 16 lanes, in all of them.
__device__ __forceinline__ float max16(float v) {
#define CCGLIB_ROTATED(n) \
  __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + n, 0xf, 0xf, true))
  v = __builtin_fmaxf(v, CCGLIB_ROTATED(8));
  v = __builtin_fmaxf(v, CCGLIB_ROTATED(4));
  v = __builtin_fmaxf(v, CCGLIB_ROTATED(2));
  v = __builtin_fmaxf(v, CCGLIB_ROTATED(1));
#undef CCGLIB_ROTATED
  return v;
}

template <int TOUT> constexpr float kTop = TOUT == kFloat8e4m3 ? 448.f : 57344.f;

// The factor of a group; `scale` as it is stored (a float's bits, or a byte).
template <int TOUT, bool E8M0> __device__ __forceinline__ float factor_of(float amax, unsigned *scale) {
  amax = __builtin_fmaxf(amax, kSmallest);
  const float s = amax / kTop<TOUT>;
  if constexpr (E8M0) {
    const unsigned byte = (__builtin_bit_cast(unsigned, s) + 0x7fffffu) >> 23;   // (the exponent, one more unless a power of two)
    *scale = byte;
    return __builtin_bit_cast(float, (254u - byte) << 23);
  } else {
    *scale = __builtin_bit_cast(unsigned, s);
    return kTop<TOUT> / amax;
  }
}

template <bool E8M0> __device__ __forceinline__ void store_scale(char *scales, size_t at, unsigned scale) {
  if constexpr (E8M0) {
    reinterpret_cast<unsigned char *>(scales)[at] = (unsigned char)scale;
  } else {
    reinterpret_cast<unsigned *>(scales)[at] = scale;
  }
}

template <int TOUT> __device__ __forceinline__ unsigned four(float a, float b, float c, float d) {
  int w = 0;
  if constexpr (TOUT == kFloat8e4m3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return (unsigned)w;
}

// Groups along the rows, no transpose, few rows: sixteen lanes to a group.
template <int TIN, int TOUT, bool E8M0>
__global__ __launch_bounds__(256) void quantize_rows(Args a) {
  using In = typename Loaded<TIN>::type;
  const unsigned id = blockIdx.x * 16 + threadIdx.x / 16;   // group
  const unsigned groups = a.tiles_n;
  const unsigned row = id / groups, g = id - row * groups;   // (row: over all matrices)
  if (row >= a.batch * a.m) return;
  const unsigned b = row / a.m, r = row - b * a.m;
  const unsigned n0 = g * kGroup + (threadIdx.x & 15) * 8;
  float v[8];
  load8<TIN>(reinterpret_cast<const In *>(a.in) + (size_t)row * a.in_pitch + n0, n0 < a.n ? (int)(a.n - n0) : 0, v);
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = __builtin_fmaxf(amax, finite_magnitude(v[e]));
  unsigned scale;
  const float f = factor_of<TOUT, E8M0>(max16(amax), &scale);
  if (n0 < a.out_pitch) {
    *reinterpret_cast<uint2_t *>(a.out + (size_t)row * a.out_pitch + n0) =
        uint2_t{four<TOUT>(v[0] * f, v[1] * f, v[2] * f, v[3] * f), four<TOUT>(v[4] * f, v[5] * f, v[6] * f, v[7] * f)};
  }
  if ((threadIdx.x & 15) == 0) store_scale<E8M0>(a.scales, ((size_t)b * groups + g) * a.scales_pitch + r, scale);
}

// Any kind of group, either or both orientations: a block has 128 x 128 values, a thread 8 x 8 of them, so that the
// values are read once and both directions' maxima come out of registers. The transposed bytes go through LDS into whole
// rows of 128.
template <int TIN, int TOUT, bool E8M0, bool BLOCKS, bool DIRECT, bool TRANSPOSED>
__global__ __launch_bounds__(256) void quantize_tile(Args a) {
  using In = typename Loaded<TIN>::type;
  constexpr int PITCH = kGroup + 16;
  __shared__ __attribute__((aligned(16))) unsigned char bytes[TRANSPOSED ? kGroup * PITCH : 16];
  __shared__ float maxima[TRANSPOSED || BLOCKS ? 4 * kGroup : 4];
  const int tid = threadIdx.x, c = tid & 15, r8 = tid >> 4, wave = tid >> 6;
  const unsigned tiles = a.tiles_m * a.tiles_n;
  const unsigned b = blockIdx.x / tiles, t = blockIdx.x - b * tiles, tm = t / a.tiles_n, tn = t - tm * a.tiles_n;
  const unsigned m0 = tm * kGroup + r8 * 8, n0 = tn * kGroup + c * 8;
  const In *in = reinterpret_cast<const In *>(a.in) + ((size_t)b * a.m + m0) * a.in_pitch + n0;
  const int valid = n0 < a.n ? (int)(a.n - n0) : 0;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) load8<TIN>(in + (size_t)i * a.in_pitch, m0 + i < a.m ? valid : 0, v[i]);

  unsigned scale;
  float block_factor = 0.f;
  if constexpr (BLOCKS) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) m = __builtin_fmaxf(m, finite_magnitude(v[i][e]));
    }
    m = max16(m);
    m = __builtin_fmaxf(m, __shfl_xor(m, 16));
    m = __builtin_fmaxf(m, __shfl_xor(m, 32));
    if ((tid & 63) == 0) maxima[wave] = m;
    __syncthreads();
    m = __builtin_fmaxf(__builtin_fmaxf(maxima[0], maxima[1]), __builtin_fmaxf(maxima[2], maxima[3]));
    block_factor = factor_of<TOUT, E8M0>(m, &scale);
    if (tid == 0) {
      if constexpr (DIRECT) store_scale<E8M0>(a.scales, ((size_t)b * a.tiles_n + tn) * a.scales_pitch + tm, scale);
      if constexpr (TRANSPOSED) store_scale<E8M0>(a.scales_t, ((size_t)b * a.tiles_m + tm) * a.scales_t_pitch + tn, scale);
    }
  }
  if constexpr (DIRECT) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float f = block_factor;
      if constexpr (!BLOCKS) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = __builtin_fmaxf(m, finite_magnitude(v[i][e]));
        f = factor_of<TOUT, E8M0>(max16(m), &scale);
        if (c == 0 && m0 + i < a.m) {
          store_scale<E8M0>(a.scales, ((size_t)b * a.tiles_n + tn) * a.scales_pitch + m0 + i, scale);
        }
      }
      if (m0 + i < a.m && n0 < a.out_pitch) {
        const float(&w)[8] = v[i];
        *reinterpret_cast<uint2_t *>(a.out + ((size_t)b * a.m + m0 + i) * a.out_pitch + n0) = uint2_t{
            four<TOUT>(w[0] * f, w[1] * f, w[2] * f, w[3] * f), four<TOUT>(w[4] * f, w[5] * f, w[6] * f, w[7] * f)};
      }
    }
  }
  if constexpr (TRANSPOSED) {
    float col[8];
    if constexpr (!BLOCKS) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = __builtin_fmaxf(m, finite_magnitude(v[i][e]));
        m = __builtin_fmaxf(m, __shfl_xor(m, 16));
        m = __builtin_fmaxf(m, __shfl_xor(m, 32));
        col[e] = m;
        if ((tid & 63) < 16) maxima[wave * kGroup + c * 8 + e] = m;
      }
      __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float f = block_factor;
      if constexpr (!BLOCKS) {
        const int at = c * 8 + e;
        const float m = __builtin_fmaxf(__builtin_fmaxf(maxima[at], maxima[kGroup + at]),
                                        __builtin_fmaxf(maxima[2 * kGroup + at], maxima[3 * kGroup + at]));
        f = factor_of<TOUT, E8M0>(m, &scale);
        if (r8 == 0 && n0 + e < a.n) {
          store_scale<E8M0>(a.scales_t, ((size_t)b * a.tiles_m + tm) * a.scales_t_pitch + n0 + e, scale);
        }
      }
      *reinterpret_cast<uint2_t *>(bytes + (c * 8 + e) * PITCH + r8 * 8) =
          uint2_t{four<TOUT>(v[0][e] * f, v[1][e] * f, v[2][e] * f, v[3][e] * f),
                  four<TOUT>(v[4][e] * f, v[5][e] * f, v[6][e] * f, v[7][e] * f)};
    }
    (void)col;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 32 + (tid >> 3), at = (tid & 7) * 16;   // (eight lanes a row)
      const unsigned n = tn * kGroup + row, m = tm * kGroup + at;
      if (n < a.n && m < a.out_t_pitch) {
        *reinterpret_cast<uint4_t *>(a.out_t + ((size_t)b * a.n + n) * a.out_t_pitch + m) =
            *reinterpret_cast<const uint4_t *>(bytes + row * PITCH + at);
      }
    }
  }
}

template <int TIN, int TOUT, bool E8M0>
hipError_t launch(const QuantizeParams &p, const Args &a, hipStream_t stream) {
  const bool direct = p.out != nullptr, transposed = p.out_t != nullptr, blocks = p.group == kScaleBlocks;
  if (direct && !transposed && !blocks) {
    const size_t groups = (size_t)p.batch * p.m * a.tiles_n;
    quantize_rows<TIN, TOUT, E8M0><<<(unsigned)ceil_div(groups, 16), 256, 0, stream>>>(a);
    return hipGetLastError();
  }
  const unsigned grid = (unsigned)((size_t)p.batch * a.tiles_m * a.tiles_n);
  if (blocks) {
    if (direct && transposed) {
      quantize_tile<TIN, TOUT, E8M0, true, true, true><<<grid, 256, 0, stream>>>(a);
    } else if (direct) {
      quantize_tile<TIN, TOUT, E8M0, true, true, false><<<grid, 256, 0, stream>>>(a);
    } else {
      quantize_tile<TIN, TOUT, E8M0, true, false, true><<<grid, 256, 0, stream>>>(a);
    }
  } else if (direct) {
    quantize_tile<TIN, TOUT, E8M0, false, true, true><<<grid, 256, 0, stream>>>(a);
  } else {
    quantize_tile<TIN, TOUT, E8M0, false, false, true><<<grid, 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <int TIN> hipError_t launch_typed(const QuantizeParams &p, const Args &a, hipStream_t stream) {
  const bool e8m0 = p.scale_type == kScaleE8m0;
  if (p.type_out == kFloat8e4m3) {
    return e8m0 ? launch<TIN, kFloat8e4m3, true>(p, a, stream) : launch<TIN, kFloat8e4m3, false>(p, a, stream);
  }
  return e8m0 ? launch<TIN, kFloat8e5m2, true>(p, a, stream) : launch<TIN, kFloat8e5m2, false>(p, a, stream);
}

}  // namespace

hipError_t launch_quantize(const QuantizeParams &p, hipStream_t stream) {
  if (p.batch == 0 || p.m == 0 || p.n == 0) return hipSuccess;
  Args a;
  a.in = static_cast<const char *>(p.in);
  a.out = static_cast<unsigned char *>(p.out);
  a.out_t = static_cast<unsigned char *>(p.out_t);
  a.scales = static_cast<char *>(p.scales);
  a.scales_t = static_cast<char *>(p.scales_t);
  a.batch = p.batch;
  a.m = p.m;
  a.n = p.n;
  a.in_pitch = p.in_pitch;
  a.out_pitch = (unsigned)scaled_pitch(p.n);
  a.out_t_pitch = (unsigned)scaled_pitch(p.m);
  a.scales_pitch = (unsigned)scaled_pitch(scale_rows(p.m, p.group));
  a.scales_t_pitch = (unsigned)scaled_pitch(scale_rows(p.n, p.group));
  a.tiles_m = (unsigned)ceil_div(p.m, kScaleGroup);
  a.tiles_n = (unsigned)ceil_div(p.n, kScaleGroup);
  switch (p.type_in) {
    case kFloat32: return launch_typed<kFloat32>(p, a, stream);
    case kFloat16: return launch_typed<kFloat16>(p, a, stream);
    default: return launch_typed<kBfloat16>(p, a, stream);
  }
}

}  // namespace ccglib_amd
