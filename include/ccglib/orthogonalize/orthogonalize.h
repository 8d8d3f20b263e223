// ccglib::orthogonalize::Orthogonalize: updates of weights made nearly orthogonal by Newton-Schulz steps (ccglib_amd.h). No
// counterpart in the reference; an inline wrapper over the C ABI.
#ifndef CCGLIB_ORTHOGONALIZE_ORTHOGONALIZE_H_
#define CCGLIB_ORTHOGONALIZE_ORTHOGONALIZE_H_

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::orthogonalize {

class Orthogonalize {
 public:
  Orthogonalize(size_t B, size_t M, size_t N, hipDevice_t &device, hipStream_t &stream, ValueType type = ValueType::bfloat16,
                int steps = 5, float a = 3.4445f, float b = -4.7750f, float c = 2.0315f, float epsilon = 1e-7f,
                size_t input_pitch = 0, size_t output_pitch = 0) {
    detail::check(ccglib_orthogonalize_create(&handle_, B, M, N, detail::ordinal(device), stream, type, steps, a, b, c, epsilon,
                                              input_pitch, output_pitch));
  }
  Orthogonalize(const Orthogonalize &) = delete;
  Orthogonalize &operator=(const Orthogonalize &) = delete;
  ~Orthogonalize() { ccglib_orthogonalize_destroy(handle_); }

  // d_output may be d_input.
  void Run(hipDeviceptr_t d_input, hipDeviceptr_t d_output) {
    detail::check(ccglib_orthogonalize_run(handle_, d_input, d_output));
  }

 private:
  ccglib_orthogonalize_t handle_ = nullptr;
};

}  // namespace ccglib::orthogonalize
#endif  // CCGLIB_ORTHOGONALIZE_ORTHOGONALIZE_H_
