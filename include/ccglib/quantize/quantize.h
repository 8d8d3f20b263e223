// ccglib::quantize::Quantize: matrices to 8 bits with a scale for each group of 128 values, as they are, transposed, or both
// (layout and formulas: ccglib_amd.h). No counterpart in the reference; an inline wrapper over the C ABI.
#ifndef CCGLIB_QUANTIZE_QUANTIZE_H_
#define CCGLIB_QUANTIZE_QUANTIZE_H_

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::quantize {

// Distance in elements of rows of n 8-bit values, and of rows of n scales.
inline size_t Pitch(size_t n) { return ccglib_scaled_pitch(n); }

class Quantize {
 public:
  Quantize(size_t B, size_t M, size_t N, hipDevice_t &device, hipStream_t &stream, ValueType input_type,
           ValueType output_type = ValueType::float8e4m3, ScaleGroup group = ScaleGroup::scale_rows,
           ScaleType scale_type = ScaleType::scale_float32, size_t input_pitch = 0) {
    detail::check(ccglib_quantize_create(&handle_, B, M, N, detail::ordinal(device), stream, input_type, output_type, group,
                                         scale_type, input_pitch));
  }
  Quantize(const Quantize &) = delete;
  Quantize &operator=(const Quantize &) = delete;
  ~Quantize() { ccglib_quantize_destroy(handle_); }

  // Either pair of outputs may be null.
  void Run(hipDeviceptr_t d_input, hipDeviceptr_t d_output, hipDeviceptr_t d_scales, hipDeviceptr_t d_output_t = nullptr,
           hipDeviceptr_t d_scales_t = nullptr) {
    detail::check(ccglib_quantize_run(handle_, d_input, d_output, d_scales, d_output_t, d_scales_t));
  }

 private:
  ccglib_quantize_t handle_ = nullptr;
};

}  // namespace ccglib::quantize
#endif  // CCGLIB_QUANTIZE_QUANTIZE_H_
