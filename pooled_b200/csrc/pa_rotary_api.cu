// C entry points of pa_rotary (include/pooled_attn.h): frequencies on the host, one launch per call.
#include <math.h>

#include <algorithm>
#include <new>

#include "pa_host.cuh"
#include "pa_params.cuh"

namespace pa {
cudaError_t launch_rotary(const RotaryParams& p, bool append, uint32_t sms, cudaStream_t st);
}
using namespace pa;

struct pa_rotary {
  pa_ctx* ctx = nullptr;
  pa_rotary_config cfg{};
  double freq[128] = {};          // radians per position
  double mscale = 1.0;
  double* turns = nullptr;        // device: freq / 2 pi
};

static constexpr double kTwoPi = 6.283185307179586476925286766559;

// the frequencies of a configuration that pa_rotary_create has checked
static void rotary_frequencies(const pa_rotary_config& c, double* f, double* mscale) {
  const double n = c.n_rot, fast = c.fast != 0.0 ? c.fast : (c.scaling == PA_ROPE_SCALE_YARN ? 32.0 : 4.0), slow = c.slow != 0.0 ? c.slow : 1.0;
  const double theta = c.scaling == PA_ROPE_SCALE_NTK ? c.theta * pow(c.factor, n / (n - 2.0)) : c.theta;
  double lo = 0.0, hi = 0.0;
  if (c.scaling == PA_ROPE_SCALE_YARN) {
    auto at = [&](double turns) { return n * log((double)c.original / (turns * kTwoPi)) / (2.0 * log(theta)); };
    lo = std::max(floor(at(fast)), 0.0);
    hi = std::min(ceil(at(slow)), n - 1.0);
  }
  for (uint32_t i = 0; i < c.n_rot / 2; ++i) {
    f[i] = pow(theta, -(2.0 * (double)i) / n);
    double kept = 1.0;            // share of the unscaled frequency
    if (c.scaling == PA_ROPE_SCALE_LINEAR) kept = 0.0;
    else if (c.scaling == PA_ROPE_SCALE_YARN) kept = 1.0 - std::min(1.0, std::max(0.0, ((double)i - lo) / std::max(hi - lo, 0.001)));
    else if (c.scaling == PA_ROPE_SCALE_BANDS) kept = std::min(1.0, std::max(0.0, ((double)c.original * f[i] / kTwoPi - slow) / (fast - slow)));
    f[i] = f[i] * kept + f[i] / c.factor * (1.0 - kept);
  }
  *mscale = c.mscale != 0.0 ? c.mscale : c.scaling == PA_ROPE_SCALE_YARN && c.factor > 1.0 ? 1.0 + 0.1 * log(c.factor) : 1.0;
}

extern "C" int pa_rotary_create(pa_ctx* ctx, const pa_rotary_config* cfg, pa_rotary** out) {
  GUARD(ctx);
  if (!cfg || !out) return fail(ctx, PA_EINVAL, "pa_rotary_create: null argument");
  *out = nullptr;
  pa_rotary_config c = *cfg;
  if (c.n_rot < 2 || (c.n_rot & 1) || c.n_rot > ctx->cfg.head_dim)
    return fail(ctx, PA_EINVAL, "pa_rotary_create: n_rot %u must be even and 2 .. head_dim %u", c.n_rot, ctx->cfg.head_dim);
  if (c.layout > PA_ROPE_INTERLEAVED || c.scaling > PA_ROPE_SCALE_BANDS) return fail(ctx, PA_EINVAL, "pa_rotary_create: unknown layout %u or scaling %u", c.layout, c.scaling);
  if (!(c.theta > 1.0) || !isfinite(c.theta)) return fail(ctx, PA_EINVAL, "pa_rotary_create: theta must be a finite number above 1");
  if (c.scaling == PA_ROPE_SCALE_NONE) c.factor = 1.0;
  else if (!(c.factor > 0.0) || !isfinite(c.factor)) return fail(ctx, PA_EINVAL, "pa_rotary_create: the scaling factor must be a finite number above 0");
  if (c.scaling == PA_ROPE_SCALE_NTK && c.n_rot < 4) return fail(ctx, PA_EINVAL, "pa_rotary_create: PA_ROPE_SCALE_NTK needs at least 4 rotated dims");
  if (!isfinite(c.mscale)) return fail(ctx, PA_EINVAL, "pa_rotary_create: mscale must be finite");
  if (c.scaling == PA_ROPE_SCALE_YARN || c.scaling == PA_ROPE_SCALE_BANDS) {
    if (c.original < 1) return fail(ctx, PA_EINVAL, "pa_rotary_create: this scaling needs the number of trained positions (original)");
    if (c.fast == 0.0) c.fast = c.scaling == PA_ROPE_SCALE_YARN ? 32.0 : 4.0;
    if (c.slow == 0.0) c.slow = 1.0;
    if (!(c.slow > 0.0) || !(c.fast > c.slow) || !isfinite(c.fast)) return fail(ctx, PA_EINVAL, "pa_rotary_create: fast must be above slow, and slow above 0");
  }
  pa_rotary* r = new (std::nothrow) pa_rotary();
  if (!r) return fail(ctx, PA_ENOMEM, "pa_rotary_create: out of host memory");
  r->ctx = ctx; r->cfg = c;
  rotary_frequencies(c, r->freq, &r->mscale);
  double turns[128];
  const uint32_t half = c.n_rot / 2;
  bool finite = isfinite((float)r->mscale);
  for (uint32_t i = 0; i < half; ++i) { turns[i] = r->freq[i] / kTwoPi; finite = finite && isfinite(turns[i] * 2147483648.0); }
  if (!finite) {
    delete r;
    return fail(ctx, PA_EINVAL, "pa_rotary_create: this scaling leaves frequencies or a factor on cos and sin that are not finite");
  }
  DeviceScope on(ctx->device);
  cudaError_t e = cudaMalloc(&r->turns, half * sizeof(double));
  if (e == cudaSuccess) e = cudaMemcpy(r->turns, turns, half * sizeof(double), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
  if (e != cudaSuccess) {
    cudaGetLastError();
    cudaFree(r->turns);
    delete r;
    return fail(ctx, e == cudaErrorMemoryAllocation ? PA_ENOMEM : PA_ECUDA, "pa_rotary_create: %s", cudaGetErrorString(e));
  }
  *out = r;
  return PA_OK;
}

extern "C" int pa_rotary_destroy(pa_rotary* r) {
  if (!r) return PA_OK;
  DeviceScope on(r->ctx->device);
  cudaFree(r->turns);
  delete r;
  return PA_OK;
}

extern "C" int pa_rotary_freqs(const pa_rotary* r, double* freqs, double* mscale) {
  if (!r) return PA_EINVAL;
  if (freqs) std::copy(r->freq, r->freq + r->cfg.n_rot / 2, freqs);
  if (mscale) *mscale = r->mscale;
  return PA_OK;
}

static uint32_t esize(int dtype) { return dtype == PA_F16 ? 2 : 4; }

extern "C" int pa_rotary_apply(pa_rotary* r, const void* x, int x_dtype, uint64_t xcs, uint64_t xhs, uint32_t n_heads, const int32_t* positions,
                               int32_t pos, uint32_t n_cols, void* y, int y_dtype, uint64_t ycs, uint64_t yhs, void* stream) {
  if (!r) return PA_EINVAL;
  pa_ctx* ctx = r->ctx;
  GUARD(ctx);
  if (!x || !y) return fail(ctx, PA_EINVAL, "pa_rotary_apply: null x or y");
  if ((x_dtype != PA_F32 && x_dtype != PA_F16) || (y_dtype != PA_F32 && y_dtype != PA_F16)) return fail(ctx, PA_EINVAL, "pa_rotary_apply: unknown dtype");
  const uint32_t hd = ctx->cfg.head_dim;
  if (n_heads < 1 || n_cols < 1 || n_heads > 65536 || n_cols > 0x7fffffffu) return fail(ctx, PA_EINVAL, "pa_rotary_apply: %u heads, %u columns", n_heads, n_cols);
  if (!positions && (int64_t)pos + n_cols - 1 > INT32_MAX) return fail(ctx, PA_EINVAL, "pa_rotary_apply: position %d + %u columns passes 2^31", pos, n_cols);
  if ((uintptr_t)x % esize(x_dtype) || (uintptr_t)y % esize(y_dtype) || ((uintptr_t)positions & 3)) return fail(ctx, PA_EINVAL, "pa_rotary_apply: a pointer is not aligned to its type");
  if (pieces_overlap(n_cols, ycs, n_heads, yhs, hd))
    return fail(ctx, PA_EINVAL, "pa_rotary_apply: heads of %u values at column stride %llu and head stride %llu of y overlap", hd, (unsigned long long)ycs, (unsigned long long)yhs);
  if (x == y && (x_dtype != y_dtype || (n_heads > 1 && xhs != yhs) || (n_cols > 1 && xcs != ycs)))
    return fail(ctx, PA_EINVAL, "pa_rotary_apply: y may be x with the same type and strides only");
  RotaryParams p{};
  p.turns = r->turns; p.mscale = (float)r->mscale; p.hd = hd; p.n_rot = r->cfg.n_rot; p.layout = r->cfg.layout; p.n_cols = n_cols;
  p.q = x; p.q_col_stride = xcs; p.q_head_stride = xhs; p.q_heads = n_heads;
  p.q_out = y; p.q_out_col_stride = ycs; p.q_out_head_stride = yhs; p.in_f16 = x_dtype == PA_F16; p.out_f16 = y_dtype == PA_F16;
  p.positions = positions; p.pos[0] = pos;
  DeviceScope on(ctx->device);
  CU_TRY(ctx, launch_rotary(p, false, (uint32_t)ctx->sm_count, (cudaStream_t)stream));
  ctx->stats.kernel_launches++; ctx->stats.calls++;
  // into a cache: what follows on that layer fetches none of its rows ahead of its wait
  const uintptr_t y0 = (uintptr_t)y, y1 = y0 + ((n_cols - 1) * ycs + (n_heads - 1) * yhs + hd) * esize(y_dtype);
  for (const pa_layer* L : ctx->layers) {
    const uint64_t bytes = (uint64_t)L->n_seqs * L->max_seq * ctx->kv_dim * (L->kv_format == PA_KV_F16 ? 2 : 4);
    for (const void* cache : {L->k ? (const void*)L->k : L->k_alt, L->v ? (const void*)L->v : L->v_alt})
      if (y0 < (uintptr_t)cache + bytes && (uintptr_t)cache < y1) { ctx->inflight_layer = L; ctx->inflight_row0 = 0; }
  }
  return PA_OK;
}

extern "C" int pa_rotary_append(pa_rotary* r, pa_layer* L, const pa_item* items, uint32_t n_items, const uint32_t* rows, const void* q, uint64_t qcs,
                                uint64_t qhs, const void* k, const void* v, uint64_t kvcs, void* q_out, int q_out_dtype, uint64_t q_out_cs, void* stream) {
  if (!r || !L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  if (r->ctx != ctx) return fail(ctx, PA_EINVAL, "pa_rotary_append: the rotation belongs to another context");
  if (L->kv_format != PA_KV_F16) return fail(ctx, PA_EUNSUPPORTED, "pa_rotary_append: f16 caches only");
  if (!items || !k || !v || (q && !q_out)) return fail(ctx, PA_EINVAL, "pa_rotary_append: null items, k, v or q_out");
  if (n_items < 1 || n_items > (uint32_t)kMaxShared) return fail(ctx, PA_EINVAL, "pa_rotary_append: 1 to %d items per call", kMaxShared);
  if (q_out_dtype != PA_F32 && q_out_dtype != PA_F16) return fail(ctx, PA_EINVAL, "pa_rotary_append: unknown q_out dtype");
  const uint32_t hd = ctx->cfg.head_dim, ae = esize((int)ctx->cfg.act_dtype);
  if ((uintptr_t)q % ae || (uintptr_t)k % ae || (uintptr_t)v % ae || (q && (uintptr_t)q_out % esize(q_out_dtype)))
    return fail(ctx, PA_EINVAL, "pa_rotary_append: a pointer is not aligned to its type");
  RotaryParams p{};
  uint64_t total = 0;
  uint32_t row_first[kMaxShared], lowest = 0xffffffffu;
  p.one_each = 1;
  for (uint32_t i = 0; i < n_items; ++i) {
    const pa_item& it = items[i];
    if (it.seq >= L->n_seqs) return fail(ctx, PA_EINVAL, "pa_rotary_append: sequence %u of %u", it.seq, L->n_seqs);
    if (it.n_cols < 1 || (uint64_t)it.pos + it.n_cols > (1ull << 31)) return fail(ctx, PA_EINVAL, "pa_rotary_append: item %u has %u columns at position %u", i, it.n_cols, it.pos);
    if (!rows && it.pos < L->origin) return fail(ctx, PA_EINVAL, "pa_rotary_append: position %u lies ahead of the layer's first, %u", it.pos, L->origin);
    const uint32_t row = rows ? rows[i] : it.pos - L->origin;
    if ((uint64_t)row + it.n_cols > L->max_seq)
      return fail(ctx, PA_EINVAL, "pa_rotary_append: rows %u..%llu pass the layer's %u", row, (unsigned long long)row + it.n_cols - 1, L->max_seq);
    for (uint32_t j = 0; j < i; ++j)
      if (items[j].seq == it.seq && row < row_first[j] + items[j].n_cols && row_first[j] < row + it.n_cols)
        return fail(ctx, PA_EINVAL, "pa_rotary_append: items %u and %u store the same row of sequence %u", j, i, it.seq);
    row_first[i] = row;
    lowest = std::min(lowest, row);
    p.pos[i] = (int32_t)it.pos; p.col0[i] = (uint32_t)total; p.row[i] = (uint64_t)it.seq * L->max_seq + row;
    if (it.n_cols != 1) p.one_each = 0;
    total += it.n_cols;
  }
  if (total > ctx->cfg.max_cols) return fail(ctx, PA_EINVAL, "pa_rotary_append: %llu columns, the context was created for at most %u", (unsigned long long)total, ctx->cfg.max_cols);
  if (q == q_out && q && ((int)ctx->cfg.act_dtype != q_out_dtype || (ctx->cfg.n_heads > 1 && qhs != hd) || (total > 1 && qcs != q_out_cs)))
    return fail(ctx, PA_EINVAL, "pa_rotary_append: q_out may be q with its type and strides only (heads packed)");
  if (q && total > 1 && q_out_cs < ctx->q_dim) return fail(ctx, PA_EINVAL, "pa_rotary_append: the column stride of q_out is below %u", ctx->q_dim);
  p.turns = r->turns; p.mscale = (float)r->mscale; p.hd = hd; p.n_rot = r->cfg.n_rot; p.layout = r->cfg.layout; p.n_cols = (uint32_t)total; p.n_items = n_items;
  p.q = q; p.q_col_stride = qcs; p.q_head_stride = qhs; p.q_heads = ctx->cfg.n_heads;
  p.q_out = q_out; p.q_out_col_stride = q_out_cs; p.q_out_head_stride = hd; p.in_f16 = ctx->cfg.act_dtype == PA_F16; p.out_f16 = q_out_dtype == PA_F16;
  p.k = k; p.v = v; p.kv_col_stride = kvcs; p.kv_heads = ctx->cfg.n_kv_heads; p.k_cache = L->k; p.v_cache = L->v;
  DeviceScope on(ctx->device);
  CU_TRY(ctx, launch_rotary(p, true, (uint32_t)ctx->sm_count, (cudaStream_t)stream));
  ctx->stats.kernel_launches++; ctx->stats.calls++;
  // what follows on this layer may start before the rows are stored: it fetches early only below the lowest of them
  if (ctx->inflight_layer == L) lowest = std::min(lowest, ctx->inflight_row0);
  ctx->inflight_layer = L; ctx->inflight_row0 = lowest;
  return PA_OK;
}
