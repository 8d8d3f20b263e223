// C++ caller of the 16-bit linear layers and of the routing between experts: small whole numbers, whose sums and products
// are exact in bfloat16 and 32 bits, so that every result is known.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <string>
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

// Whole numbers from -1 to 1.
static std::vector<float> whole_numbers(size_t n, unsigned seed) {
  std::vector<float> v(n);
  for (float &x : v) {
    seed = seed * 1664525u + 1013904223u;
    x = (float)((int)(seed >> 24) % 3 - 1);
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

// y = relu(x W^T + b) + r and its gradients. (Sums of at most 96 products: no more than 8 bits.)
static void fused(hipDevice_t device, hipStream_t stream) {
  const size_t M = 90, N = 70, K = 96;
  const std::vector<float> x = whole_numbers(M * K, 1), w = whole_numbers(N * K, 2), b = whole_numbers(N, 3), r = whole_numbers(M * N, 4),
                           dy = whole_numbers(M * N, 5);
  Buffer<uint16_t> d_x(to_bfloat16(x)), d_w(to_bfloat16(w)), d_b(to_bfloat16(b)), d_r(to_bfloat16(r)), d_dy(to_bfloat16(dy)), d_y(M * N),
      d_z(M * N), d_dx(M * K);
  Buffer<float> d_dw(N * K), d_db(N);
  ccglib::pipeline::FusedLinear layer(M, N, K, device, stream, ccglib::bfloat16, ccglib::activation_relu);
  layer.Forward(d_x.ptr(), d_w.ptr(), d_b.ptr(), d_r.ptr(), d_y.ptr(), d_z.ptr());
  layer.Backward(d_dy.ptr(), d_z.ptr(), d_x.ptr(), d_w.ptr(), d_dx.ptr(), d_dw.ptr(), d_db.ptr());
  const std::vector<uint16_t> y = d_y.host(stream), dx = d_dx.host(stream);
  const std::vector<float> dw = d_dw.host(stream), db = d_db.host(stream);
  CHECK(layer.KernelName(1).find("input") != std::string::npos);
  std::vector<float> dz(M * N);
  bool ok = true;
  for (size_t m = 0; m < M; ++m) {
    for (size_t n = 0; n < N; ++n) {
      float z = b[n];
      for (size_t k = 0; k < K; ++k) z += x[m * K + k] * w[n * K + k];
      ok = ok && value_of(y[m * N + n]) == (z > 0 ? z : 0) + r[m * N + n];
      dz[m * N + n] = z > 0 ? dy[m * N + n] : 0;
    }
  }
  CHECK(ok);
  for (size_t m = 0; m < M; ++m) {
    for (size_t k = 0; k < K; ++k) {
      float want = 0;
      for (size_t n = 0; n < N; ++n) want += dz[m * N + n] * w[n * K + k];
      ok = ok && value_of(dx[m * K + k]) == want;
    }
  }
  CHECK(ok);
  for (size_t n = 0; n < N; ++n) {
    float sum = 0;
    for (size_t m = 0; m < M; ++m) sum += dz[m * N + n];
    ok = ok && db[n] == sum;
    for (size_t k = 0; k < K; ++k) {
      float want = 0;
      for (size_t m = 0; m < M; ++m) want += dz[m * N + n] * x[m * K + k];
      ok = ok && dw[n * K + k] == want;
    }
  }
  CHECK(ok);
}

// Tokens to one of two experts each by their logits, through it, and back with a weight of 1.
static void experts(hipDevice_t device, hipStream_t stream) {
  const size_t T = 100, E = 3, N = 40, K = 50;
  std::vector<float> logits(T * E, 0.f);
  for (size_t t = 0; t < T; ++t) logits[t * E + (t % 3 ? 2 : 0)] = 5.f;    // (nobody chooses the second one)
  const std::vector<float> x = whole_numbers(T * K, 6), w = whole_numbers(E * N * K, 7);
  Buffer<float> d_logits(logits), d_weights(T), d_dweights(std::vector<float>(T, 1.f)), d_dlogits(T * E);
  Buffer<int> d_experts(T), d_offsets(E + 1), d_slots(T);
  Buffer<uint16_t> d_x(to_bfloat16(x)), d_w(to_bfloat16(w)), d_xs(T * K), d_ys(T * N), d_out(T * N);
  ccglib::route::Route route(T, E, 1, device, stream);
  ccglib::route::Combine spread(T, 1, K, device, stream), combine(T, 1, N, device, stream);
  ccglib::pipeline::GroupedLinear layer(E, T, N, K, device, stream, ccglib::bfloat16, ccglib::activation_none, ccglib::float32, false);
  route.Run(d_logits.ptr(), d_experts.ptr(), d_weights.ptr(), d_offsets.ptr(), d_slots.ptr());
  spread.Spread(d_x.ptr(), d_slots.ptr(), nullptr, d_xs.ptr());
  layer.Forward(d_xs.ptr(), d_offsets.ptr(), d_w.ptr(), nullptr, nullptr, d_ys.ptr());
  combine.Run(d_ys.ptr(), d_slots.ptr(), d_weights.ptr(), d_out.ptr());
  route.Backward(d_logits.ptr(), d_experts.ptr(), d_weights.ptr(), d_dweights.ptr(), d_dlogits.ptr());
  const std::vector<uint16_t> out = d_out.host(stream);
  const std::vector<int> offsets = d_offsets.host(stream);
  const std::vector<float> dlogits = d_dlogits.host(stream);
  CHECK(offsets[0] == 0 && offsets[1] == 34 && offsets[2] == 34 && offsets[3] == 100);
  bool ok = true;
  for (size_t t = 0; t < T; ++t) {
    const size_t e = t % 3 ? 2 : 0;
    for (size_t n = 0; n < N; ++n) {
      float want = 0;
      for (size_t k = 0; k < K; ++k) want += x[t * K + k] * w[(e * N + n) * K + k];
      ok = ok && value_of(out[t * N + n]) == want;
    }
  }
  for (float d : dlogits) ok = ok && d == 0.f;      // (a softmax of one: its weight is 1, whatever the logit)
  CHECK(ok);
}

static void refusals(hipDevice_t device, hipStream_t stream) {
  bool refused = false;
  try {
    ccglib::pipeline::FusedLinear layer(8, 8, 8, device, stream, ccglib::float32);
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
  fused(device, stream);
  experts(device, stream);
  refusals(device, stream);
  HIP(hipStreamDestroy(stream));
  if (failures == 0) std::printf("all checks passed\n");
  return failures != 0;
}
