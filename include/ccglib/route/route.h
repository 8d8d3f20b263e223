// ccglib::route::Route: which k of E experts each token goes to, with what weights, and where its rows lie when all are
// sorted by expert; ccglib::route::Combine: rows spread to those places and summed back (formulas: ccglib_amd.h). No
// counterpart in the reference; inline wrappers over the C ABI.
#ifndef CCGLIB_ROUTE_ROUTE_H_
#define CCGLIB_ROUTE_ROUTE_H_

#include <hip/hip_runtime.h>

#include <ccglib/common/error.h>
#include <ccglib/common/types.h>

namespace ccglib::route {

class Route {
 public:
  Route(size_t T, size_t E, size_t k, hipDevice_t &device, hipStream_t &stream, ValueType type = ValueType::float32,
        bool normalize = true) {
    detail::check(ccglib_route_create(&handle_, T, E, k, detail::ordinal(device), stream, type, normalize));
  }
  Route(const Route &) = delete;
  Route &operator=(const Route &) = delete;
  ~Route() { ccglib_route_destroy(handle_); }

  void Run(hipDeviceptr_t d_logits, hipDeviceptr_t d_experts, hipDeviceptr_t d_weights, hipDeviceptr_t d_offsets,
           hipDeviceptr_t d_slots) {
    detail::check(ccglib_route_run(handle_, d_logits, d_experts, d_weights, d_offsets, d_slots));
  }
  // With what Run wrote; d_logits may be null with normalize.
  void Backward(hipDeviceptr_t d_logits, hipDeviceptr_t d_experts, hipDeviceptr_t d_weights, hipDeviceptr_t d_dweights,
                hipDeviceptr_t d_dlogits) {
    detail::check(ccglib_route_backward(handle_, d_logits, d_experts, d_weights, d_dweights, d_dlogits));
  }

 private:
  ccglib_route_t handle_ = nullptr;
};

class Combine {
 public:
  Combine(size_t T, size_t k, size_t N, hipDevice_t &device, hipStream_t &stream, ValueType type = ValueType::bfloat16,
          size_t rows = 0, size_t y_pitch = 0, size_t out_pitch = 0) {
    detail::check(ccglib_combine_create(&handle_, T, k, N, detail::ordinal(device), stream, type, rows, y_pitch, out_pitch));
  }
  Combine(const Combine &) = delete;
  Combine &operator=(const Combine &) = delete;
  ~Combine() { ccglib_combine_destroy(handle_); }

  // d_weights may be null (all 1), here and below.
  void Run(hipDeviceptr_t d_y, hipDeviceptr_t d_slots, hipDeviceptr_t d_weights, hipDeviceptr_t d_out) {
    detail::check(ccglib_combine_run(handle_, d_y, d_slots, d_weights, d_out));
  }
  void Spread(hipDeviceptr_t d_x, hipDeviceptr_t d_slots, hipDeviceptr_t d_weights, hipDeviceptr_t d_y) {
    detail::check(ccglib_combine_spread(handle_, d_x, d_slots, d_weights, d_y));
  }
  // Of Run; a gradient that is not wanted is null.
  void Backward(hipDeviceptr_t d_dout, hipDeviceptr_t d_y, hipDeviceptr_t d_slots, hipDeviceptr_t d_weights, hipDeviceptr_t d_dy,
                hipDeviceptr_t d_dweights = nullptr) {
    detail::check(ccglib_combine_backward(handle_, d_dout, d_y, d_slots, d_weights, d_dy, d_dweights));
  }

 private:
  ccglib_combine_t handle_ = nullptr;
};

}  // namespace ccglib::route
#endif  // CCGLIB_ROUTE_ROUTE_H_
