// ccglib::mma::ScaledGEMM: C (+)= A B^T of 8-bit operands with a scale for each group of 128 along K (layout and formula:
// ccglib_amd.h). No counterpart in the reference; an inline wrapper over the C ABI.
#ifndef CCGLIB_GEMM_SCALED_GEMM_H_
#define CCGLIB_GEMM_SCALED_GEMM_H_

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::mma {

class ScaledGEMM {
 public:
  ScaledGEMM(size_t B, size_t M, size_t N, size_t K, hipDevice_t &device, hipStream_t &stream,
             ValueType a_type = ValueType::float8e4m3, ValueType b_type = ValueType::float8e4m3,
             ValueType c_type = ValueType::bfloat16, ScaleGroup a_group = ScaleGroup::scale_rows,
             ScaleGroup b_group = ScaleGroup::scale_blocks, ScaleType scale_type = ScaleType::scale_float32,
             bool accumulate = false, size_t pitch_a = 0, size_t pitch_b = 0, size_t pitch_c = 0) {
    detail::check(ccglib_scaled_gemm_create(&handle_, B, M, N, K, detail::ordinal(device), stream, a_type, b_type, c_type,
                                            a_group, b_group, scale_type, accumulate, pitch_a, pitch_b, pitch_c));
  }
  ScaledGEMM(const ScaledGEMM &) = delete;
  ScaledGEMM &operator=(const ScaledGEMM &) = delete;
  ~ScaledGEMM() { ccglib_scaled_gemm_destroy(handle_); }

  void Run(hipDeviceptr_t d_a, hipDeviceptr_t d_scales_a, hipDeviceptr_t d_b, hipDeviceptr_t d_scales_b, hipDeviceptr_t d_c) {
    detail::check(ccglib_scaled_gemm_run(handle_, d_a, d_scales_a, d_b, d_scales_b, d_c));
  }

 private:
  ccglib_scaled_gemm_t handle_ = nullptr;
};

}  // namespace ccglib::mma
#endif  // CCGLIB_GEMM_SCALED_GEMM_H_
