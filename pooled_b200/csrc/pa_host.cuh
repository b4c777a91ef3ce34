// What the files with C entry points share: error messages, the guards of a call, the current device, the sizes of a context's buffers.
#pragma once
#include <algorithm>

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

// How many records, one (o, m, l) per (query row, run of tiles), the partial buffers of a context hold and a call may use.
inline void size_records(pa_ctx* ctx) {
  const size_t rows = (size_t)ctx->cfg.max_cols * ctx->cfg.n_heads;
  // about 64 rows x one CTA per SM; the split planner keeps every call inside this capacity
  ctx->part_slots = 16384;
  // a prefill call of few columns splits its keys: 400 columns of 24 heads three ways are 28800 records
  ctx->pf_slots = std::max<size_t>(ctx->part_slots, std::min<size_t>(32768, rows * kPrefillSplits));
  // Trees: one for each of 64 rows of two CTAs an SM, or 136 for each row of max_cols tokens, which are runs of 4 tiles (the shortest that f32 outputs
  // ask for) behind 34816 committed rows, up to 32768 in all; more tokens: four for each row, up to 65536.  (32768 for every context were 14 MB more at
  // head_dim 256 for one of 8 columns and 16 heads, and no other plan for its trees.)
  const size_t few = std::max<size_t>(rows * 136, (size_t)ctx->sm_count * 128);
  ctx->tree_slots = std::max(ctx->pf_slots, std::min(few, std::max<size_t>(32768, std::min<size_t>(65536, rows * 4))));
}

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
