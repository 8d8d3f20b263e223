// ccglib::pipeline::GroupedLinear: FusedLinear with a weight matrix for each of E experts, on rows that are sorted by
// expert (formulas: ccglib_amd.h). No counterpart in the reference; an inline wrapper over the C ABI.
#ifndef CCGLIB_PIPELINE_GROUPED_LINEAR_H_
#define CCGLIB_PIPELINE_GROUPED_LINEAR_H_

#include <string>

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::pipeline {

class GroupedLinear {
 public:
  GroupedLinear(size_t E, size_t M, size_t N, size_t K, hipDevice_t &device, hipStream_t &stream,
                ValueType type = ValueType::bfloat16, Activation activation = Activation::activation_none,
                ValueType gradient_type = ValueType::float32, bool training = true, size_t x_pitch = 0, size_t w_pitch = 0,
                size_t y_pitch = 0) {
    detail::check(ccglib_grouped_linear_create(&handle_, E, M, N, K, detail::ordinal(device), stream, type, activation,
                                               gradient_type, training, x_pitch, w_pitch, y_pitch));
  }
  GroupedLinear(const GroupedLinear &) = delete;
  GroupedLinear &operator=(const GroupedLinear &) = delete;
  ~GroupedLinear() { ccglib_grouped_linear_destroy(handle_); }

  // d_offsets: E + 1 int32 on the device. d_bias, d_residual and d_z may be null.
  void Forward(hipDeviceptr_t d_x, hipDeviceptr_t d_offsets, hipDeviceptr_t d_w, hipDeviceptr_t d_bias, hipDeviceptr_t d_residual,
               hipDeviceptr_t d_y, hipDeviceptr_t d_z = nullptr) {
    detail::check(ccglib_grouped_linear_forward(handle_, d_x, d_offsets, d_w, d_bias, d_residual, d_y, d_z));
  }
  // Gradients that are not wanted are null; without an activation d_z may be null too.
  void Backward(hipDeviceptr_t d_dy, hipDeviceptr_t d_z, hipDeviceptr_t d_x, hipDeviceptr_t d_offsets, hipDeviceptr_t d_w,
                hipDeviceptr_t d_dx, hipDeviceptr_t d_dw, hipDeviceptr_t d_dbias = nullptr, bool accumulate = false) {
    detail::check(ccglib_grouped_linear_backward(handle_, d_dy, d_z, d_x, d_offsets, d_w, d_dx, d_dw, d_dbias, accumulate));
  }
  // Which kernel computes y (0), dx (1), dW (2).
  std::string KernelName(int product = 0) const {
    char name[160];
    detail::check(ccglib_grouped_linear_kernel_name(handle_, product, name, sizeof name));
    return name;
  }

 private:
  ccglib_grouped_linear_t handle_ = nullptr;
};

}  // namespace ccglib::pipeline
#endif  // CCGLIB_PIPELINE_GROUPED_LINEAR_H_
