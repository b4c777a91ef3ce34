// What the files with C entry points share: error messages, the guards of a call, the current device.
#pragma once
#include "pa_common.cuh"

namespace pa {

// sets the message pa_last_error() gives (ctx == nullptr: for failures before a context exists) and returns `code`
int fail(pa_ctx* ctx, int code, const char* fmt, ...) __attribute__((format(printf, 3, 4)));

// the calling thread's current device for the length of a call
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
    if (before_ != device) cudaSetDevice(device);
    device_ = device;
  }
  ~DeviceScope() { if (before_ != device_) cudaSetDevice(before_); }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = 0, device_ = 0;
};

}  // namespace pa

#define CU_TRY(ctx, expr)                                                                         \
  do {                                                                                            \
    cudaError_t e_ = (expr);                                                                      \
    if (e_ != cudaSuccess) {                                                                      \
      (ctx)->failed = true;                                                                       \
      return fail((ctx), PA_ECUDA, "%s failed: %s", #expr, cudaGetErrorString(e_));               \
    }                                                                                             \
  } while (0)

#define GUARD(ctx)                                                                                       \
  do {                                                                                                   \
    if (!(ctx)) return PA_EINVAL;                                                                        \
    if ((ctx)->failed) return fail((ctx), PA_ESTATE, "an earlier step failed (%s); call pa_reset() first", (ctx)->err.c_str()); \
  } while (0)
