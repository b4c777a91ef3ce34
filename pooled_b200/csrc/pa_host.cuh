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

// whether any two of the pieces of `len` values that begin at c * col_stride + h * head_stride, c < n_cols, h < n_heads, overlap
inline bool pieces_overlap(uint64_t n_cols, uint64_t col_stride, uint64_t n_heads, uint64_t head_stride, uint64_t len) {
  typedef unsigned __int128 wide;
  if ((n_cols > 1 && col_stride < len) || (n_heads > 1 && head_stride < len)) return true;
  if (n_cols < 2 || n_heads < 2 || col_stride >= (wide)(n_heads - 1) * head_stride + len || head_stride >= (wide)(n_cols - 1) * col_stride + len) return false;
  for (uint64_t h = 1; h < n_heads; ++h) {                  // h heads on, and the columns next to that distance
    const wide at = (wide)h * head_stride;
    for (wide c = at / col_stride, last = c + 1; c <= last && c < n_cols; ++c)
      if ((c * col_stride > at ? c * col_stride - at : at - c * col_stride) < len) return true;
  }
  return false;
}

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
