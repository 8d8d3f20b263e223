// Host-side helpers of the C entry points: the last error's text, the device a call works on, what a device and a
// stream must be.
#ifndef CCGLIB_AMD_HOST_UTIL_H_
#define CCGLIB_AMD_HOST_UTIL_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ccglib_amd.h"

namespace ccglib_amd {

// Keeps the text for ccglib_last_error of this thread; returns `code`.
int fail(int code, const char *fmt, ...);
int fail_hip(hipError_t e, const char *what);

#define HIP_TRY(expr)                                   \
  do {                                                  \
    hipError_t e_ = (expr);                             \
    if (e_ != hipSuccess) return fail_hip(e_, #expr);   \
  } while (0)

// Makes `device` current for the lifetime of the guard.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    if (hipGetDevice(&previous_) != hipSuccess) previous_ = -1;
    if (previous_ != device) {
      status_ = hipSetDevice(device);
      switched_ = (status_ == hipSuccess);
    }
  }
  ~DeviceGuard() {
    if (switched_ && previous_ >= 0) (void)hipSetDevice(previous_);
  }
  hipError_t status() const { return status_; }

 private:
  int previous_ = -1;
  bool switched_ = false;
  hipError_t status_ = hipSuccess;
};

// Whether the ordinal names a gfx950 device.
int check_device(int device);

// Device memory of an object.
struct Buffer {
  void *p = nullptr;
  ~Buffer() {
    if (p) (void)hipFree(p);
  }
  char *at(size_t offset) const { return static_cast<char *>(p) + offset; }
};

// Allocates `bytes` and clears the first `zeroed`; the memory is cleared when the call returns.
inline int allocate(Buffer *b, size_t bytes, size_t zeroed) {
  if (bytes == 0) return CCGLIB_OK;
  HIP_TRY(hipMalloc(&b->p, bytes));
  if (zeroed) {
    HIP_TRY(hipMemset(b->p, 0, zeroed));
    HIP_TRY(hipStreamSynchronize(nullptr));
  }
  return CCGLIB_OK;
}

inline bool aligned(const void *p, size_t to) { return (uintptr_t)p % to == 0; }

}  // namespace ccglib_amd
#endif  // CCGLIB_AMD_HOST_UTIL_H_
