// Conversion to 8 bits with a scale for each group of 128 values of a row, or of 128 x 128 values; of a matrix, of its
// transpose, or of both in one pass over it. With t the largest value of the type:
//   amax = max(2^-100, largest finite |x| of the group)
//   float32 scales:  scale = amax / t, factor = t / amax   (each rounded once, to 32 bits)
//   e8m0 scales:     scale = 2^ceil(log2(amax / t)), factor = 1 / scale
//   q = 8-bit value nearest to x * factor, ties to even; NaN stays NaN, infinity stays infinity or, in e4m3, is NaN
// Values that are not finite leave the scale of their group alone. Cannot do without 2 or 4 bytes in and 1 or 2 out a value.
#include <algorithm>
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

// Eight neighbours of a row as they lie in memory: 16-bit types take two to a register, so that more waves fit.
template <int TYPE> struct Eight {
  static constexpr int WORDS = TYPE == kFloat32 ? 8 : 4;
  unsigned w[WORDS];

  __device__ __forceinline__ void load(const typename Loaded<TYPE>::type *p) {
#pragma unroll
    for (int h = 0; h < WORDS / 4; ++h) {
      const uint4_unaligned_t got = reinterpret_cast<const uint4_unaligned_t *>(p)[h];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * h + e] = got[e];
    }
  }

  // From p on, of which `valid` are there; the others are zero.
  __device__ __forceinline__ void load_some(const typename Loaded<TYPE>::type *p, int valid) {
#pragma unroll
    for (int e = 0; e < WORDS; ++e) {
      if constexpr (TYPE == kFloat32) {
        w[e] = e < valid ? reinterpret_cast<const unsigned *>(p)[e] : 0;
      } else {
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
        const unsigned lo = 2 * e < valid ? q[2 * e] : 0, hi = 2 * e + 1 < valid ? q[2 * e + 1] : 0;
        w[e] = lo | hi << 16;
      }
    }
  }

  // Without the first n values (of 0 to 8), zeros behind the others.
  __device__ __forceinline__ void drop(int n) {
    constexpr int EACH = 8 / WORDS;
    if constexpr (EACH == 2) {
#pragma unroll
      for (int e = 0; e < WORDS; ++e) w[e] = n & 1 ? w[e] >> 16 | (e + 1 < WORDS ? w[e + 1] << 16 : 0) : w[e];
    }
#pragma unroll
    for (int by = 1; by <= WORDS; by *= 2) {
#pragma unroll
      for (int e = 0; e < WORDS; ++e) w[e] = n & by * EACH ? (e + by < WORDS ? w[e + by] : 0) : w[e];
    }
  }

  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (TYPE == kFloat32) {
      const unsigned x = w[e];
      return __builtin_bit_cast(float, x);
    } else if constexpr (TYPE == kBfloat16) {
      return __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    } else {
      return (float)__builtin_bit_cast(_Float16, (unsigned short)(e % 2 ? w[e / 2] >> 16 : w[e / 2]));
    }
  }

  // Here and later the values are made of the words, not kept.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int e = 0; e < WORDS; ++e) asm volatile("" : "+v"(w[e]));
  }
};

// Values n0 to n0 + 7 of R rows, of which `rows` are there (perhaps none) and have n values; `first`: the first one of them, behind
// another row if there is none. Where a wave is not whole, its lanes read the row's last eight and the last row instead and
// drop what they are not for: no lane waits for another's branch.
template <int TYPE, int R>
__device__ __forceinline__ void load_rows(const typename Loaded<TYPE>::type *first, size_t pitch, int rows, unsigned n0, unsigned n,
                                          Eight<TYPE> (&v)[R]) {
  if (__all(rows >= R && n0 + 8 <= n)) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i].load(first + (ptrdiff_t)i * (ptrdiff_t)pitch + n0);
  } else if (n >= 8) {
    const unsigned from = n0 < n - 8 ? n0 : n - 8, behind = n0 - from < 8 ? n0 - from : 8;
#pragma unroll
    for (int i = 0; i < R; ++i) v[i].load(first + (ptrdiff_t)(i < rows ? i : rows - 1) * (ptrdiff_t)pitch + from);
#pragma unroll
    for (int i = 0; i < R; ++i) v[i].drop(i < rows ? (int)behind : 8);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i].load_some(first + (ptrdiff_t)i * (ptrdiff_t)pitch + n0, i < rows && n0 < n ? (int)(n - n0) : 0);
  }
}

// Magnitudes are compared as the integers that their bits are, in 16-bit types two at a time; infinity and NaN are the
// largest ones.
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
template <int TYPE> constexpr unsigned kInfinite = TYPE == kFloat32 ? 0x7f800000u : TYPE == kFloat16 ? 0x7c00u : 0x7f80u;

__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }

template <int TYPE> __device__ __forceinline__ unsigned larger_of_word(unsigned a, unsigned b) {
  if constexpr (TYPE == kFloat32) return larger(a, b);
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
}

// Magnitudes of a word's values; FINITE: of those that are finite, the others zero.
template <int TYPE, bool FINITE> __device__ __forceinline__ unsigned magnitudes(unsigned w) {
  if constexpr (TYPE == kFloat32) {
    const unsigned m = w & 0x7fffffffu;
    return FINITE && m >= kInfinite<TYPE> ? 0 : m;
  } else {
    const unsigned m = w & 0x7fff7fffu;
    if constexpr (!FINITE) return m;
    return ((m & 0xffffu) < kInfinite<TYPE> ? m & 0xffffu : 0) | (m >> 16 < kInfinite<TYPE> ? m & 0xffff0000u : 0);
  }
}

// The larger magnitude of a word; a magnitude as a float.
template <int TYPE> __device__ __forceinline__ unsigned larger_in(unsigned w) {
  if constexpr (TYPE == kFloat32) return w;
  return larger(w & 0xffffu, w >> 16);
}
template <int TYPE> __device__ __forceinline__ float as_float(unsigned m) {
  if constexpr (TYPE == kFloat32) return __builtin_bit_cast(float, m);
  if constexpr (TYPE == kBfloat16) return __builtin_bit_cast(float, m << 16);
  return (float)__builtin_bit_cast(_Float16, (unsigned short)m);
}

// Lane l of each 16 gets the value of lane f(l) of these 16.
template <int CONTROL> __device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kXor7 = 0x141, kRotate = 0x120, kBroadcast = 0x150;

// Maximum over each 16 lanes, in all of them.
__device__ __forceinline__ unsigned max16(unsigned v) {
  v = larger(v, dpp<kRotate + 8>(v));
  v = larger(v, dpp<kRotate + 4>(v));
  v = larger(v, dpp<kRotate + 2>(v));
  return larger(v, dpp<kRotate + 1>(v));
}

// Maximum of v[l % 8] over each 16 lanes, in lane l: halves are handed over and kept in turn.
__device__ __forceinline__ unsigned max16_of_eight(const unsigned (&v)[8], int l) {
  unsigned four[4], two[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) four[j] = larger((l & 4) ? v[j + 4] : v[j], dpp<kXor7>((l & 4) ? v[j] : v[j + 4]));
#pragma unroll
  for (int j = 0; j < 2; ++j) two[j] = larger((l & 2) ? four[j + 2] : four[j], dpp<kXor2>((l & 2) ? four[j] : four[j + 2]));
  const unsigned one = larger((l & 1) ? two[1] : two[0], dpp<kXor1>((l & 1) ? two[0] : two[1]));
  return larger(one, dpp<kRotate + 8>(one));
}

// Lane l of each 16 holds the value of row l % 8: all eight in each lane.
__device__ __forceinline__ void spread(float v, float (&all)[8]) {
  const unsigned bits = __builtin_bit_cast(unsigned, v);
  unsigned got[8] = {dpp<kBroadcast>(bits),     dpp<kBroadcast + 1>(bits), dpp<kBroadcast + 2>(bits), dpp<kBroadcast + 3>(bits),
                     dpp<kBroadcast + 4>(bits), dpp<kBroadcast + 5>(bits), dpp<kBroadcast + 6>(bits), dpp<kBroadcast + 7>(bits)};
#pragma unroll
  for (int i = 0; i < 8; ++i) all[i] = __builtin_bit_cast(float, got[i]);
}

// Maxima of v over the four lanes l, l ^ 16, l ^ 32, l ^ 48; two of the eight stay in each of them: v[4 h + 2 q] and the
// next, for l = 32 h + 16 q.
__device__ __forceinline__ uint2_t max4_of_eight(const unsigned (&v)[8]) {
  unsigned four[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto got = __builtin_amdgcn_permlane32_swap(v[j], v[j + 4], false, false);
    four[j] = larger(got[0], got[1]);
  }
  const auto a = __builtin_amdgcn_permlane16_swap(four[0], four[2], false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(four[1], four[3], false, false);
  return uint2_t{larger(a[0], a[1]), larger(b[0], b[1])};
}

// Largest magnitudes of the rows and columns of 8 x 8 values.
template <int TYPE, bool FINITE>
__device__ __forceinline__ void maxima_of(const Eight<TYPE> (&v)[8], unsigned (&rows)[8], unsigned (&columns)[8]) {
  constexpr int WORDS = Eight<TYPE>::WORDS;
  unsigned words[WORDS] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned row = 0;
#pragma unroll
    for (int e = 0; e < WORDS; ++e) {
      const unsigned m = magnitudes<TYPE, FINITE>(v[i].w[e]);
      row = larger_of_word<TYPE>(row, m);
      words[e] = larger_of_word<TYPE>(words[e], m);
    }
    rows[i] = larger_in<TYPE>(row);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) columns[e] = WORDS == 8 ? words[e % WORDS] : e % 2 ? words[e / 2] >> 16 : words[e / 2] & 0xffffu;
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

// Groups along the rows, no transpose: sixteen lanes to a group, so that one row already spreads over the chip. One row of 4096
// bf16: 2.0 us, a round trip.
template <int TIN, int TOUT, bool E8M0>
__global__ __launch_bounds__(256) void quantize_rows(Args a) {
  using In = typename Loaded<TIN>::type;
  const unsigned id = blockIdx.x * 16 + threadIdx.x / 16;   // group
  const unsigned groups = a.tiles_n;
  const unsigned row = id / groups, g = id - row * groups;   // (row: over all matrices)
  if (row >= a.batch * a.m) return;
  const unsigned b = row / a.m, r = row - b * a.m;
  const unsigned n0 = g * kGroup + (threadIdx.x & 15) * 8;
  Eight<TIN> rows[1], &v = rows[0];
  load_rows<TIN, 1>(reinterpret_cast<const In *>(a.in) + (size_t)row * a.in_pitch, a.in_pitch, 1, n0, a.n, rows);
  unsigned amax = 0;
#pragma unroll
  for (int e = 0; e < v.WORDS; ++e) amax = larger_of_word<TIN>(amax, magnitudes<TIN, true>(v.w[e]));
  unsigned scale;
  const float f = factor_of<TOUT, E8M0>(as_float<TIN>(max16(larger_in<TIN>(amax))), &scale);
  if (n0 < a.out_pitch) {
    *reinterpret_cast<uint2_t *>(a.out + (size_t)row * a.out_pitch + n0) =
        uint2_t{four<TOUT>(v[0] * f, v[1] * f, v[2] * f, v[3] * f), four<TOUT>(v[4] * f, v[5] * f, v[6] * f, v[7] * f)};
  }
  if ((threadIdx.x & 15) == 0) store_scale<E8M0>(a.scales, ((size_t)b * groups + g) * a.scales_pitch + r, scale);
}

// Any kind of group, either or both orientations: a block has 128 x 128 values, a thread 8 x 8 of them, so that the
// values are read once and both directions' maxima come out of registers. A group's factor is made by one lane, and the
// transposed bytes go through LDS into whole rows of 128. Blocks follow one another on the same XCD, as their rows' ends
// share lines of its L2. 8192 x 8192 bf16 rows, both ways: 62 us, 4.4 TB/s,
// where a copy reaches 4.9 and a transpose alone 5.8 (8191 x 8200, whose rows share lines: 65 to 70 us; 4096 x 4096 in blocks: 16).
template <int TIN, int TOUT, bool E8M0, bool BLOCKS, bool DIRECT, bool TRANSPOSED>
__global__ __launch_bounds__(256) void quantize_tile(Args a) {
  using In = typename Loaded<TIN>::type;
  constexpr int PITCH = kGroup + 16;
  __shared__ __attribute__((aligned(16))) unsigned char bytes[TRANSPOSED ? kGroup * PITCH : 16];
  __shared__ __attribute__((aligned(16))) unsigned maxima[TRANSPOSED || BLOCKS ? 4 * kGroup : 4];
  __shared__ __attribute__((aligned(16))) float factors[TRANSPOSED && !BLOCKS ? kGroup : 4];
  const int tid = threadIdx.x, c = tid & 15, r8 = tid >> 4, wave = tid >> 6;
  const unsigned id = blockIdx.x & 7, part = gridDim.x / 8, rest = gridDim.x & 7;   // (block k runs on XCD k % 8)
  const unsigned tiles = a.tiles_m * a.tiles_n, tile = id * part + (id < rest ? id : rest) + blockIdx.x / 8;
  const unsigned b = tile / tiles, t = tile - b * tiles, tm = t / a.tiles_n, tn = t - tm * a.tiles_n;
  const unsigned m0 = tm * kGroup + r8 * 8, n0 = tn * kGroup + c * 8;
  const In *in = reinterpret_cast<const In *>(a.in) + ((size_t)b * a.m + m0) * a.in_pitch;
  Eight<TIN> v[8];
  load_rows<TIN, 8>(in, a.in_pitch, (int)(a.m - m0), n0, a.n, v);

  unsigned rows[8], columns[8], all = 0;
  maxima_of<TIN, false>(v, rows, columns);
#pragma unroll
  for (int i = 0; i < 8; ++i) all = larger(all, rows[i]);
  if (__builtin_expect(__any(all >= kInfinite<TIN>), 0)) {
    maxima_of<TIN, true>(v, rows, columns);
    all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) all = larger(all, rows[i]);
  }

  unsigned scale;
  float row_factors[8], column_factors[8];
  if constexpr (BLOCKS) {
    all = max16(all);
    all = larger(all, __shfl_xor(all, 16));
    all = larger(all, __shfl_xor(all, 32));
    if ((tid & 63) == 0) maxima[wave] = all;
    __syncthreads();
    const unsigned m = larger(larger(maxima[0], maxima[1]), larger(maxima[2], maxima[3]));
    const float f = factor_of<TOUT, E8M0>(as_float<TIN>(m), &scale);
    if (tid == 0) {
      if constexpr (DIRECT) store_scale<E8M0>(a.scales, ((size_t)b * a.tiles_n + tn) * a.scales_pitch + tm, scale);
      if constexpr (TRANSPOSED) store_scale<E8M0>(a.scales_t, ((size_t)b * a.tiles_m + tm) * a.scales_t_pitch + tn, scale);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) row_factors[i] = column_factors[i] = f;
  } else {
    if constexpr (TRANSPOSED) {
      const int lane = tid & 63;
      *reinterpret_cast<uint2_t *>(maxima + wave * kGroup + c * 8 + (lane >> 4) * 2) = max4_of_eight(columns);
    }
    if constexpr (DIRECT) {
      const float f = factor_of<TOUT, E8M0>(as_float<TIN>(max16_of_eight(rows, c)), &scale);
      const unsigned m = m0 + c;
      if (c < 8 && m < a.m) store_scale<E8M0>(a.scales, ((size_t)b * a.tiles_n + tn) * a.scales_pitch + m, scale);
      spread(f, row_factors);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i].forget();
  if constexpr (DIRECT) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (m0 + i < a.m && n0 < a.out_pitch) {
        const Eight<TIN> &w = v[i];
        const float f = row_factors[i];
        *reinterpret_cast<uint2_t *>(a.out + ((size_t)b * a.m + m0 + i) * a.out_pitch + n0) = uint2_t{
            four<TOUT>(w[0] * f, w[1] * f, w[2] * f, w[3] * f), four<TOUT>(w[4] * f, w[5] * f, w[6] * f, w[7] * f)};
      }
    }
  }
  if constexpr (TRANSPOSED) {
    if constexpr (!BLOCKS) {
      __syncthreads();
      if (tid < kGroup) {
        const unsigned m = larger(larger(maxima[tid], maxima[kGroup + tid]), larger(maxima[2 * kGroup + tid], maxima[3 * kGroup + tid]));
        factors[tid] = factor_of<TOUT, E8M0>(as_float<TIN>(m), &scale);
        const unsigned n = tn * kGroup + tid;
        if (n < a.n) store_scale<E8M0>(a.scales_t, ((size_t)b * a.tiles_m + tm) * a.scales_t_pitch + n, scale);
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) column_factors[e] = factors[c * 8 + e];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].forget();
    // (16-byte pieces of a row lie at places XORed with bits of the row, so that a wave's writes meet every bank)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = column_factors[e];
      *reinterpret_cast<uint2_t *>(bytes + (c * 8 + e) * PITCH + (r8 ^ (c & 14)) * 8) =
          uint2_t{four<TOUT>(v[0][e] * f, v[1][e] * f, v[2][e] * f, v[3][e] * f),
                  four<TOUT>(v[4][e] * f, v[5][e] * f, v[6][e] * f, v[7][e] * f)};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 32 + (tid >> 3), at = (tid & 7) * 16;   // (eight lanes a row)
      const unsigned n = tn * kGroup + row, m = tm * kGroup + at;
      if (n < a.n && m < a.out_t_pitch) {
        *reinterpret_cast<uint4_t *>(a.out_t + ((size_t)b * a.n + n) * a.out_t_pitch + m) =
            *reinterpret_cast<const uint4_t *>(bytes + row * PITCH + (at ^ ((row >> 4) << 4)));
      }
    }
  }
}

template <int TIN, int TOUT, bool E8M0>
hipError_t launch(const QuantizeParams &p, const Args &a, unsigned grid, hipStream_t stream) {
  const bool direct = p.out != nullptr, transposed = p.out_t != nullptr, blocks = p.group == kScaleBlocks;
  if (direct && !transposed && !blocks) {
    quantize_rows<TIN, TOUT, E8M0><<<grid, 256, 0, stream>>>(a);
  } else if (blocks) {
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

template <int TIN> hipError_t launch_typed(const QuantizeParams &p, const Args &a, unsigned grid, hipStream_t stream) {
  const bool e8m0 = p.scale_type == kScaleE8m0;
  if (p.type_out == kFloat8e4m3) {
    return e8m0 ? launch<TIN, kFloat8e4m3, true>(p, a, grid, stream) : launch<TIN, kFloat8e4m3, false>(p, a, grid, stream);
  }
  return e8m0 ? launch<TIN, kFloat8e5m2, true>(p, a, grid, stream) : launch<TIN, kFloat8e5m2, false>(p, a, grid, stream);
}

hipError_t launch_part(const QuantizeParams &p, const Args &a, size_t grid, hipStream_t stream) {
  switch (p.type_in) {
    case kFloat32: return launch_typed<kFloat32>(p, a, (unsigned)grid, stream);
    case kFloat16: return launch_typed<kFloat16>(p, a, (unsigned)grid, stream);
    default: return launch_typed<kBfloat16>(p, a, (unsigned)grid, stream);
  }
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

  // A launch of 2^32 work-items or more is no error to the runtime, but starts what is left of the number modulo 2^32: as many
  // matrices at a time as one takes, or as many rows of a matrix.
  constexpr size_t kMost = 0xffffffffu / 256;
  const bool rows_only = p.out && !p.out_t && p.group == kScaleRows;
  const size_t each = rows_only ? (size_t)p.m * a.tiles_n : (size_t)a.tiles_m * a.tiles_n;   // groups, or tiles, of a matrix
  const size_t most = rows_only ? kMost * 16 : kMost;
  if (!rows_only && each > most) return hipErrorInvalidValue;                                // (no card holds that many values)
  const size_t matrices = std::max<size_t>(1, most / each), rows = each <= most ? p.m : most / a.tiles_n;
  const size_t in_size = (size_t)p.in_pitch * bits_of(p.type_in) / 8, scale = p.scale_type == kScaleE8m0 ? 1 : 4;
  for (size_t b = 0; b < p.batch; b += matrices) {
    for (size_t r = 0; r < p.m; r += rows) {
      Args part = a;
      part.batch = (unsigned)std::min<size_t>(matrices, p.batch - b);
      part.m = (unsigned)std::min<size_t>(rows, p.m - r);
      part.in += (b * p.m + r) * in_size;
      if (a.out) {
        part.out += (b * p.m + r) * a.out_pitch;
        part.scales += (b * a.tiles_n * a.scales_pitch + r) * scale;
      }
      if (a.out_t) {
        part.out_t += b * p.n * a.out_t_pitch;
        part.scales_t += b * a.tiles_m * a.scales_t_pitch * scale;
      }
      const size_t grid = rows_only ? ceil_div((size_t)part.batch * part.m * a.tiles_n, 16) : part.batch * each;
      if (const hipError_t e = launch_part(p, part, grid, stream)) return e;
    }
  }
  return hipSuccess;
}

}  // namespace ccglib_amd
