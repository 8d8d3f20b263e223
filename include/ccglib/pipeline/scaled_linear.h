// ccglib::pipeline::ScaledLinear: a linear layer, y = x W^T, forward and backward, by products of 8-bit copies that the
// object makes and keeps (ccglib_amd.h). No counterpart in the reference; an inline wrapper over the C ABI.
#ifndef CCGLIB_PIPELINE_SCALED_LINEAR_H_
#define CCGLIB_PIPELINE_SCALED_LINEAR_H_

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::pipeline {

class ScaledLinear {
 public:
  ScaledLinear(size_t M, size_t N, size_t K, hipDevice_t &device, hipStream_t &stream, ValueType type = ValueType::bfloat16,
               ValueType gradient_type = ValueType::float8e5m2, ScaleType scale_type = ScaleType::scale_float32,
               bool training = true) {
    detail::check(ccglib_scaled_linear_create(&handle_, M, N, K, detail::ordinal(device), stream, type, gradient_type, scale_type,
                                              training));
  }
  ScaledLinear(const ScaledLinear &) = delete;
  ScaledLinear &operator=(const ScaledLinear &) = delete;
  ~ScaledLinear() { ccglib_scaled_linear_destroy(handle_); }

  void SetWeights(hipDeviceptr_t d_w) { detail::check(ccglib_scaled_linear_set_weights(handle_, d_w)); }
  void Forward(hipDeviceptr_t d_x, hipDeviceptr_t d_y) { detail::check(ccglib_scaled_linear_forward(handle_, d_x, d_y)); }
  // With the x and W of the last Forward (after another SetWeights d_dx is refused until the next one). d_dx or d_dw may be null.
  void Backward(hipDeviceptr_t d_dy, hipDeviceptr_t d_dx, hipDeviceptr_t d_dw, bool accumulate_dw = false) {
    detail::check(ccglib_scaled_linear_backward(handle_, d_dy, d_dx, d_dw, accumulate_dw));
  }

 private:
  ccglib_scaled_linear_t handle_ = nullptr;
};

}  // namespace ccglib::pipeline
#endif  // CCGLIB_PIPELINE_SCALED_LINEAR_H_
