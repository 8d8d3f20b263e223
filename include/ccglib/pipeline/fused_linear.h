// ccglib::pipeline::FusedLinear: a linear layer of 16-bit values with bias, activation and residual, forward and backward
// (formulas: ccglib_amd.h). No counterpart in the reference; an inline wrapper over the C ABI.
#ifndef CCGLIB_PIPELINE_FUSED_LINEAR_H_
#define CCGLIB_PIPELINE_FUSED_LINEAR_H_

#include <string>

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::pipeline {

class FusedLinear {
 public:
  FusedLinear(size_t M, size_t N, size_t K, hipDevice_t &device, hipStream_t &stream, ValueType type = ValueType::bfloat16,
              Activation activation = Activation::activation_none, ValueType gradient_type = ValueType::float32, bool training = true,
              size_t x_pitch = 0, size_t w_pitch = 0, size_t y_pitch = 0) {
    detail::check(ccglib_fused_linear_create(&handle_, M, N, K, detail::ordinal(device), stream, type, activation, gradient_type,
                                             training, x_pitch, w_pitch, y_pitch));
  }
  FusedLinear(const FusedLinear &) = delete;
  FusedLinear &operator=(const FusedLinear &) = delete;
  ~FusedLinear() { ccglib_fused_linear_destroy(handle_); }

  // d_bias, d_residual and d_z may be null; d_y may be d_residual.
  void Forward(hipDeviceptr_t d_x, hipDeviceptr_t d_w, hipDeviceptr_t d_bias, hipDeviceptr_t d_residual, hipDeviceptr_t d_y,
               hipDeviceptr_t d_z = nullptr) {
    detail::check(ccglib_fused_linear_forward(handle_, d_x, d_w, d_bias, d_residual, d_y, d_z));
  }
  // Gradients that are not wanted are null; without an activation d_z may be null too.
  void Backward(hipDeviceptr_t d_dy, hipDeviceptr_t d_z, hipDeviceptr_t d_x, hipDeviceptr_t d_w, hipDeviceptr_t d_dx,
                hipDeviceptr_t d_dw, hipDeviceptr_t d_dbias = nullptr, bool accumulate = false) {
    detail::check(ccglib_fused_linear_backward(handle_, d_dy, d_z, d_x, d_w, d_dx, d_dw, d_dbias, accumulate));
  }
  // Which kernel computes y (0), dx (1), dW (2).
  std::string KernelName(int product = 0) const {
    char name[160];
    detail::check(ccglib_fused_linear_kernel_name(handle_, product, name, sizeof name));
    return name;
  }

 private:
  ccglib_fused_linear_t handle_ = nullptr;
};

}  // namespace ccglib::pipeline
#endif  // CCGLIB_PIPELINE_FUSED_LINEAR_H_
