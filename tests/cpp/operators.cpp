// C++ caller of the 8-bit operators with block scales and of the orthogonalised updates, on inputs whose results are
// known: small whole numbers, with a value of 448 (the largest of float8e4m3, so a scale of 1) in each group of 128.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <vector>

#include <hip/hip_runtime.h>

#include <ccglib/ccglib.hpp>

static int failures = 0;
#define CHECK(cond)                                                 \
  do {                                                              \
    if (!(cond)) {                                                  \
      ++failures;                                                   \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
    }                                                               \
  } while (0)
#define HIP(x)                                                                           \
  do {                                                                                   \
    hipError_t e_ = (x);                                                                 \
    if (e_ != hipSuccess) {                                                              \
      std::printf("HIP error %s at %s:%d\n", hipGetErrorString(e_), __FILE__, __LINE__); \
      std::exit(2);                                                                      \
    }                                                                                    \
  } while (0)

template <typename T> class Buffer {
 public:
  explicit Buffer(size_t n) : n_(n) { HIP(hipMalloc(&ptr_, n * sizeof(T))); }
  explicit Buffer(const std::vector<T> &v) : Buffer(v.size()) {
    HIP(hipMemcpy(ptr_, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice));
  }
  Buffer(const Buffer &) = delete;
  ~Buffer() { (void)hipFree(ptr_); }
  hipDeviceptr_t ptr() const { return reinterpret_cast<hipDeviceptr_t>(ptr_); }
  std::vector<T> host(hipStream_t stream) const {
    HIP(hipStreamSynchronize(stream));
    std::vector<T> v(n_);
    HIP(hipMemcpy(v.data(), ptr_, n_ * sizeof(T), hipMemcpyDeviceToHost));
    return v;
  }

 private:
  T *ptr_ = nullptr;
  size_t n_;
};

static std::vector<float> whole_numbers(size_t rows, size_t columns, unsigned seed) {
  std::vector<float> v(rows * columns);
  for (size_t r = 0; r < rows; ++r) {
    for (size_t c = 0; c < columns; ++c) {
      seed = seed * 1664525u + 1013904223u;
      v[r * columns + c] = r % 128 == c % 128 ? 448.f : (float)((int)(seed >> 24) % 5 - 2);
    }
  }
  return v;
}

static std::vector<uint16_t> to_bfloat16(const std::vector<float> &v) {   // (whole numbers of at most 8 bits)
  std::vector<uint16_t> r(v.size());
  for (size_t i = 0; i < v.size(); ++i) {
    uint32_t bits;
    __builtin_memcpy(&bits, &v[i], 4);
    r[i] = (uint16_t)(bits >> 16);
  }
  return r;
}

static float value_of(uint16_t bits) {
  const uint32_t wide = (uint32_t)bits << 16;
  float f;
  __builtin_memcpy(&f, &wide, 4);
  return f;
}

static void quantized_product(hipDevice_t device, hipStream_t stream) {
  const size_t M = 128, N = 256, K = 384;
  const std::vector<float> a = whole_numbers(M, K, 1), b = whole_numbers(N, K, 2);
  const size_t pitch = ccglib::quantize::Pitch(K);
  Buffer<float> d_a(a), d_b(b), d_sa(K / 128 * ccglib::quantize::Pitch(M)), d_sb(K / 128 * ccglib::quantize::Pitch(N / 128));
  Buffer<uint8_t> d_qa(M * pitch), d_qb(N * pitch);
  Buffer<float> d_c(M * N);
  ccglib::quantize::Quantize rows(1, M, K, device, stream, ccglib::float32);
  ccglib::quantize::Quantize blocks(1, N, K, device, stream, ccglib::float32, ccglib::float8e4m3, ccglib::scale_blocks);
  ccglib::mma::ScaledGEMM product(1, M, N, K, device, stream, ccglib::float8e4m3, ccglib::float8e4m3, ccglib::float32);
  rows.Run(d_a.ptr(), d_qa.ptr(), d_sa.ptr());
  blocks.Run(d_b.ptr(), d_qb.ptr(), d_sb.ptr());
  product.Run(d_qa.ptr(), d_sa.ptr(), d_qb.ptr(), d_sb.ptr(), d_c.ptr());
  const std::vector<float> c = d_c.host(stream);
  bool same = true;
  for (size_t m = 0; m < M; ++m) {
    for (size_t n = 0; n < N; ++n) {
      double want = 0;
      for (size_t k = 0; k < K; ++k) want += (double)a[m * K + k] * b[n * K + k];
      same = same && c[m * N + n] == (float)want;
    }
  }
  CHECK(same);
}

static void linear(hipDevice_t device, hipStream_t stream) {
  const size_t M = 256, N = 128, K = 256;
  const std::vector<float> x = whole_numbers(M, K, 3), w = whole_numbers(N, K, 4), dy = whole_numbers(M, N, 5);
  Buffer<uint16_t> d_x(to_bfloat16(x)), d_w(to_bfloat16(w)), d_dy(to_bfloat16(dy)), d_y(M * N), d_dx(M * K);
  Buffer<float> d_dw(N * K);
  ccglib::pipeline::ScaledLinear layer(M, N, K, device, stream, ccglib::bfloat16, ccglib::float8e4m3);
  layer.SetWeights(d_w.ptr());
  layer.Forward(d_x.ptr(), d_y.ptr());
  layer.Backward(d_dy.ptr(), d_dx.ptr(), d_dw.ptr());
  const std::vector<uint16_t> y = d_y.host(stream), dx = d_dx.host(stream);
  const std::vector<float> dw = d_dw.host(stream);
  // (bf16 results: half a unit is 2^-9 of the value; the sums behind them are good to 2^-13 of their largest product)
  const double near = 1.0 / 256, slack = 448.0 * 448.0 * 2 / 8192;
  bool ok = true;
  for (size_t m = 0; m < M; ++m) {
    for (size_t n = 0; n < N; ++n) {
      double want = 0;
      for (size_t k = 0; k < K; ++k) want += (double)x[m * K + k] * w[n * K + k];
      ok = ok && std::fabs(value_of(y[m * N + n]) - want) <= near * std::fabs(want) + slack;
    }
  }
  CHECK(ok);
  for (size_t m = 0; m < M; ++m) {
    for (size_t k = 0; k < K; ++k) {
      double want = 0;
      for (size_t n = 0; n < N; ++n) want += (double)dy[m * N + n] * w[n * K + k];
      ok = ok && std::fabs(value_of(dx[m * K + k]) - want) <= near * std::fabs(want) + slack;
    }
  }
  CHECK(ok);
  for (size_t n = 0; n < N; ++n) {
    for (size_t k = 0; k < K; ++k) {
      double want = 0;
      for (size_t m = 0; m < M; ++m) want += (double)dy[m * N + n] * x[m * K + k];
      ok = ok && dw[n * K + k] == (float)want;
    }
  }
  CHECK(ok);
}

// A multiple of the identity stays one; its factor runs through the steps by itself.
static void orthogonalize(hipDevice_t device, hipStream_t stream, size_t n) {
  std::vector<float> g(n * n, 0.f);
  for (size_t i = 0; i < n; ++i) g[i * n + i] = -3.f;
  Buffer<float> d_g(g), d_o(n * n);
  ccglib::orthogonalize::Orthogonalize op(1, n, n, device, stream, ccglib::float32);
  op.Run(d_g.ptr(), d_o.ptr());
  const std::vector<float> o = d_o.host(stream);
  double x = -1.0 / std::sqrt((double)n);
  for (int i = 0; i < 5; ++i) x = x * (3.4445 + x * x * (-4.7750 + 2.0315 * x * x));
  bool ok = true;
  for (size_t r = 0; r < n; ++r) {
    for (size_t c = 0; c < n; ++c) ok = ok && std::fabs(o[r * n + c] - (r == c ? x : 0.0)) < 1e-5;
  }
  CHECK(ok);
}

static void refusals(hipDevice_t device, hipStream_t stream) {
  bool refused = false;
  try {
    ccglib::quantize::Quantize q(1, 8, 8, device, stream, ccglib::int1);
  } catch (const std::runtime_error &) {
    refused = true;
  }
  CHECK(refused);
}

int main() {
  HIP(hipSetDevice(0));
  hipDevice_t device;
  HIP(hipDeviceGet(&device, 0));
  hipStream_t stream;
  HIP(hipStreamCreate(&stream));
  quantized_product(device, stream);
  linear(device, stream);
  orthogonalize(device, stream, 50);
  orthogonalize(device, stream, 300);
  refusals(device, stream);
  HIP(hipStreamDestroy(stream));
  if (failures == 0) std::printf("all checks passed\n");
  return failures != 0;
}
