// C entry points of the shared-prefix and the weighing decode, and of the eviction (include/pooled_attn.h): checks, the plan of
// the units, launches.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "pa_host.cuh"
#include "pa_params.cuh"

namespace pa {
cudaError_t launch_shared(const SharedParams& p, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& k, const CUtensorMap& v, uint32_t hd, uint32_t n_kv,
                          int dev, cudaStream_t st);
cudaError_t launch_shared_finish(const SharedFinishParams& p, uint32_t hd, uint32_t sum_ctas, cudaStream_t st);
cudaError_t launch_evict(const EvictParams& p, uint32_t sms, int dev, cudaStream_t st);
}  // namespace pa
using namespace pa;

static uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }
static uint32_t pad64(uint32_t rows) { return (rows + 63) & ~63u; }
static uint64_t scores_of(const pa_ctx* ctx, uint32_t rows) { return (uint64_t)ctx->cfg.n_heads * pad64(rows); }

// What a call's units cost, in us on the device (a model of measurements: a unit of T tiles takes T * tile + start; start: launch, q, the first
// scores, the record).  tile: 0.75 at head_dim 256 (the tensor cores), 0.8 below, two CTAs an SM; of wide units 1.17.  A record ahead of a
// unit's last one: 3 of 64 query rows.
struct UnitCost { float p_tile, p_start, p_record, o_tile, o_start; };
static UnitCost unit_cost(uint32_t hd, bool wide, uint32_t p_rows) {
  const float tile = hd == 256 ? 0.75f : 0.8f;
  return UnitCost{wide ? 1.17f : tile, wide ? 10.5f : 5.5f, 3.f * (float)p_rows / 64, tile, 5.5f};
}
// f16 outputs: the tensor cores' rounding towards zero (2^-24 of the sum at each of four additions a tile, of
// wide units eight) stays below 2^-15 of the result (2^-14)
static constexpr uint32_t kF16Tiles = 128;
// f32 outputs: most tiles of a run where records run short (1.8e-6 of the result, as 32 tiles cost 2.3e-6); runs of 16 there, that is two of 9 for
// one of 17 or 18, took 32 items behind 32768 rows (16/2 heads of 256) from 49 to 57 us
static constexpr uint32_t kF32Run = 24;
// tiles of a record for a unit of T: at most `cap`, the unit's shared out evenly
static uint32_t record_tiles(uint32_t T, uint32_t cap) { return ceil_div(T, ceil_div(T, cap)); }

// Tiles per unit (T) and the time the call takes with them.  The units run one CTA an SM at a time (two of head_dim 128 and 64), in the grid's order: the shared
// rows' units, all equal, then those of own rows, which fill what the last wave of the others leaves.  Tried: every number of splits
// of the longest of the shared rows and the items' own (beyond 24 in steps of 4 %).  Between narrow and wide units this chooses within 1.2 % of
// the faster on average over 168 calls (12 to 128 items of 6 or 8 heads, 1 to 65536 shared and 40 to 777 own rows), 12 of them more
// than 5 % off and the worst 28 % (34 items of 6 heads behind 700 rows, own rows up to 777: 31.5 us, wide 24.7).
static uint32_t plan_units(const pa_ctx* ctx, const uint32_t* rows, uint32_t n_items, uint32_t p_tiles, uint32_t row_tiles, const UnitCost& c, uint32_t cap, uint32_t most_records,
                           float* us) {
  const uint32_t n_kv = ctx->cfg.n_kv_heads;
  const float sms = (float)(ctx->sm_count * (ctx->cfg.head_dim == 256 ? 1 : 2));      // CTAs at a time
  float tiles[kMaxShared], own_tiles = 0.f, own_longest = 0.f;
  for (uint32_t i = 0; i < n_items; ++i) {
    tiles[i] = (float)ceil_div(rows[i], 64);
    own_tiles += tiles[i]; own_longest = std::max(own_longest, tiles[i]);
  }
  const uint32_t longest = std::max(1u, std::max(p_tiles, (uint32_t)own_longest));
  const uint32_t most_splits = std::min(longest, std::min(most_records, 4 * (uint32_t)ctx->sm_count));
  const float hbm = ((float)p_tiles + own_tiles) * n_kv * (float)(ctx->cfg.head_dim * 256) / 6.0e6f;      // us for its bytes
  uint32_t best = longest;
  *us = 3.0e38f;
  for (uint32_t n = 1; n <= most_splits; n += 1 + n / 24) {
    const uint32_t T = ceil_div(longest, n);
    // records of a row: the shared rows' and the longest item's
    if (ceil_div(p_tiles, T) + ceil_div((uint32_t)own_longest, T) > most_records) break;
    const uint32_t p_do = std::min(T, p_tiles), records = p_do ? ceil_div(p_do, record_tiles(T, cap)) : 1;       // of a unit of shared rows
    const float inv = 1.0f / (float)T, tp = (float)p_do * c.p_tile + c.p_start + (float)(records - 1) * c.p_record;
    const float to = std::min((float)T, own_longest) * c.o_tile + c.o_start;
    float own_units = 0.f;
    for (uint32_t i = 0; i < n_items; ++i) own_units += (float)(int)(tiles[i] * inv + 0.999f);
    own_units *= n_kv;
    const float p_units = (float)(row_tiles * ceil_div(p_tiles, T) * n_kv), waves = floorf(p_units / sms), rest = p_units - waves * sms;
    const float own_work = own_tiles * n_kv * c.o_tile + own_units * c.o_start;
    float time = (waves + (rest > 0.f ? 1.f : 0.f)) * tp;            // the shared rows
    if (own_units > 0.f) {
      if (own_units <= sms - rest) time = std::max(time, waves * tp + to);
      else {                                                         // sms - rest SMs from the last full wave on, the others a wave later
        float level = waves * tp + own_work / (sms - rest + 1.0e-3f);
        if (rest > 0.f && level > (waves + 1.f) * tp) level = (waves + 1.f) * tp + (own_work - (sms - rest) * tp) / sms;
        time = std::max(time, level + 0.5f * to);
      }
    }
    time = std::max(time, hbm + c.o_start) + 0.05f * time;           // (bound by HBM, the smaller T: more CTAs stream)
    if (time < *us) { *us = time; best = T; }
  }
  return best;
}

struct SharedCall {
  const char* who;
  pa_layer* L;
  pa_layer* prefix;             // nullptr: own rows only
  uint32_t prefix_seq, prefix_len, own_row0;
  const void* q; int q_f16; uint64_t qcs, qhs;
  const void* gate; uint64_t gcs, ghs;
  void* out; uint64_t ocs;
  bool sums;
};

// one launch of each kernel for items [first, first + n) with these own rows
static int shared_launch(const SharedCall& c, const pa_item* items, const uint32_t* rows, uint32_t first, uint32_t n, cudaStream_t st) {
  pa_layer* L = c.L;
  pa_ctx* ctx = L->ctx;
  const uint32_t hd = ctx->cfg.head_dim, nH = ctx->cfg.n_heads, n_kv = ctx->cfg.n_kv_heads, G = ctx->G;
  SharedParams p{};
  SharedFinishParams f{};
  p.n_items = n; p.n_heads = nH; p.G = G; p.max_seq = L->max_seq; p.err = ctx->dev_err;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
  const size_t aes = ctx->cfg.act_dtype == PA_F16 ? 2 : 4;
  p.q = reinterpret_cast<const uint8_t*>(c.q) + (uint64_t)first * c.qcs * (c.q_f16 ? 2 : 4); p.q_f16 = c.q_f16; p.q_col_stride = c.qcs; p.q_head_stride = c.qhs;
  p.part_o = ctx->part_o; p.part_ml = ctx->part_ml;
  const uint32_t p_tiles = c.prefix ? ceil_div(c.prefix_len, 64) : 0;
  const uint32_t most = (uint32_t)std::min<size_t>(512, ctx->pf_slots / ((size_t)n * nH));
  // row tiles of the shared rows: of 64 query rows, or of 128 where that promises less time
  p.items_per_tile = 64 / G; p.row_tiles = ceil_div(n, p.items_per_tile);
  float us = 0.f, wide_us = 0.f;
  const uint32_t cap = ctx->cfg.act_dtype == PA_F16 ? kF16Tiles : p.row_tiles > 1 && p_tiles ? 16u : 4u;
  uint32_t T = plan_units(ctx, rows + first, n, p_tiles, p.row_tiles, unit_cost(hd, false, std::min(n, p.items_per_tile) * G), cap, most, &us);
  if (hd == 256 && p_tiles && p.row_tiles > 1 && c.q_f16 && ctx->cfg.act_dtype == PA_F16 && ctx->tune.shared_wide != 0) {
    const uint32_t tiles128 = ceil_div(n, 128 / G), T128 = plan_units(ctx, rows + first, n, p_tiles, tiles128, unit_cost(hd, true, 128), kF16Tiles, most, &wide_us);
    if (wide_us < us || ctx->tune.shared_wide == 1) { p.wide = 1; p.items_per_tile = 128 / G; p.row_tiles = tiles128; T = T128; }
  }
  // tiles of a record: those of a unit of up to kF16Tiles, with f32 outputs at most four (which HBM hides), sixteen where the tensor cores
  // bound it: a unit's shared out evenly (17 as two of 9, not as one of 16 and a unit of 32: 13 items behind 11633 rows, 24/4 heads, 37 us
  // for 23).  Where that is more records than there is room for, a record is of more, and past kF32Run tiles (f16: kF16Tiles) it adds up
  // several runs.
  uint32_t own_longest = 0;
  for (uint32_t i = 0; i < n; ++i) own_longest = std::max(own_longest, ceil_div(rows[first + i], 64));
  uint32_t records = ceil_div(T, cap);
  while (records > 1 && ceil_div(p_tiles, ceil_div(T, records)) + ceil_div(own_longest, ceil_div(T, records)) > most) --records;
  uint32_t rec = ceil_div(T, records);
  p.fold = ceil_div(rec, std::max(cap, kF32Run));
  rec = ceil_div(rec, p.fold) * p.fold;
  T = records * rec;
  p.seg = rec / p.fold;
  if (c.prefix) { p.p_row0 = c.prefix_seq * c.prefix->max_seq; p.p_rows = c.prefix_len; p.p_tps = T; p.p_splits = ceil_div(p_tiles, T); }
  p.p_recs = ceil_div(p_tiles, rec);
  p.tps = T; p.own_row0 = c.own_row0;
  uint32_t units = p.p_splits * p.row_tiles;
  uint64_t floats = 0;
  for (uint32_t i = 0; i < n; ++i) {
    const uint32_t r = rows[first + i], tiles = ceil_div(r, 64);
    p.seq[i] = f.seq[i] = items[first + i].seq; p.rows[i] = f.rows[i] = r; p.cta0[i] = units; f.n_own[i] = (uint16_t)ceil_div(tiles, rec);
    p.score0[i] = f.score0[i] = floats;
    floats += scores_of(ctx, r);
    units += ceil_div(tiles, T);
  }
  p.cta0[n] = units; p.units = units;
  p.n_rec = p.p_recs + ceil_div(own_longest, rec);
  if (c.sums) p.scores = ctx->scores;
  f.part_o = p.part_o; f.part_ml = p.part_ml; f.n_rec = p.n_rec; f.p_recs = p.p_recs; f.n_items = n; f.n_heads = nH; f.G = G; f.n_kv = n_kv;
  f.gate = c.gate ? reinterpret_cast<const uint8_t*>(c.gate) + (uint64_t)first * c.gcs * aes : nullptr; f.gate_col_stride = c.gcs; f.gate_head_stride = c.ghs;
  f.out = reinterpret_cast<uint8_t*>(c.out) + (uint64_t)first * c.ocs * aes; f.out_col_stride = c.ocs; f.act_f16 = ctx->cfg.act_dtype == PA_F16;
  // few rows of many records: their dims are shared out among CTAs, else a CTA takes a row
  f.lanes = (uint64_t)n * nH * 2 <= (uint64_t)ctx->sm_count * 4 && p.n_rec > 16 ? 16 : hd / 4;
  f.merge_ctas = n * nH * (hd / 4 / f.lanes);
  uint32_t sum_ctas = 0;
  if (c.sums) {
    f.scores = ctx->scores; f.sums = L->sums; f.scale_log2 = p.scale_log2; f.max_seq = L->max_seq;
    uint8_t last[kMaxShared];            // of each lead: its last item so far
    for (uint32_t i = 0; i < n; ++i) {
      f.next[i] = 255;
      uint32_t l = 0;
      while (l < f.n_leads && f.seq[f.lead[l]] != f.seq[i]) ++l;
      if (l == f.n_leads) { f.lead[l] = (uint8_t)i; f.n_leads++; } else f.next[last[l]] = (uint8_t)i;
      last[l] = (uint8_t)i;
    }
    for (uint32_t l = 0; l < f.n_leads; ++l) {
      uint32_t longest = 0;
      for (uint32_t i = f.lead[l]; i != 255; i = f.next[i]) longest = std::max(longest, f.rows[i]);
      f.sum0[l] = sum_ctas;
      sum_ctas += n_kv * ceil_div(longest, kSumRows);
    }
    f.sum0[f.n_leads] = sum_ctas;
  }
  const pa_layer* P = c.prefix ? c.prefix : L;
  CU_TRY(ctx, launch_shared(p, P->tm_k64, P->tm_v64, L->tm_k64, L->tm_v64, hd, n_kv, ctx->device, st));
  CU_TRY(ctx, launch_shared_finish(f, hd, sum_ctas, st));
  ctx->stats.kernel_launches += 2;
  uint64_t read = c.prefix ? c.prefix_len : 0;
  for (uint32_t i = 0; i < n; ++i) read += p.rows[i];
  ctx->stats.kv_bytes_streamed += read * ctx->kv_dim * 4;
  return PA_OK;
}

static int shared_impl(const SharedCall& c, const pa_item* items, uint32_t n_items, const uint32_t* rows, cudaStream_t st) {
  pa_ctx* ctx = c.L->ctx;
  const uint64_t am = c.q_f16 ? 7 : 3;
  if ((c.qcs & am) || (c.qhs & am) || ((uintptr_t)c.q & 15)) return fail(ctx, PA_EINVAL, "%s: q strides must be multiples of 16 bytes and q 16-byte aligned", c.who);
  const uint32_t ae = ctx->cfg.act_dtype == PA_F16 ? 2 : 4;
  if ((uintptr_t)c.gate % ae || (uintptr_t)c.out % ae) return fail(ctx, PA_EINVAL, "%s: a pointer is not aligned to its type", c.who);
  if (n_items > 1 && c.ocs < ctx->q_dim) return fail(ctx, PA_EINVAL, "%s: the column stride of out is below %u", c.who, ctx->q_dim);
  DeviceScope on(ctx->device);
  // items that fit the records (two a row at least) and the room for scores go in one launch
  const uint32_t by_records = std::max<uint32_t>(1, (uint32_t)(ctx->pf_slots / (2 * (size_t)ctx->cfg.n_heads)));
  for (uint32_t i = 0; i < n_items;) {
    uint32_t n = 0;
    uint64_t floats = 0;
    while (i + n < n_items && n < by_records) {
      floats += c.sums ? scores_of(ctx, rows[i + n]) : 0;
      if (floats > ctx->scores_floats && c.sums && n) break;
      ++n;
    }
    if (int rc = shared_launch(c, items, rows, i, n, st)) return rc;
    i += n;
  }
  ctx->stats.calls++;
  ctx->inflight_layer = nullptr;         // these kernels wait for everything before them and write no cache row
  return PA_OK;
}

// what both decodes want of the layer and the items
static int shared_checks(pa_layer* L, const pa_item* items, uint32_t n_items, const void* q, int q_dtype, const void* out, const char* who) {
  pa_ctx* ctx = L->ctx;
  if (L->kv_format != PA_KV_F16) return fail(ctx, PA_EUNSUPPORTED, "%s: f16 caches only", who);
  if (L->origin) return fail(ctx, PA_EUNSUPPORTED, "%s: not on a shard of longer sequences", who);
  if (ctx->G > 64) return fail(ctx, PA_EUNSUPPORTED, "%s: more than 64 query heads per kv head", who);
  if ((size_t)ctx->cfg.n_heads * 2 > ctx->pf_slots) return fail(ctx, PA_EUNSUPPORTED, "%s: more than %zu query heads", who, ctx->pf_slots / 2);
  if (!items || !q || !out) return fail(ctx, PA_EINVAL, "%s: null items, q or out", who);
  if (q_dtype != PA_F32 && q_dtype != PA_F16) return fail(ctx, PA_EINVAL, "%s: unknown q dtype", who);
  if (n_items < 1 || n_items > (uint32_t)kMaxShared) return fail(ctx, PA_EINVAL, "%s: 1 to %d items per call", who, kMaxShared);
  for (uint32_t i = 0; i < n_items; ++i) {
    if (items[i].n_cols != 1) return fail(ctx, PA_EINVAL, "%s: item %u has %u columns; one token per item", who, i, items[i].n_cols);
    if (items[i].seq >= L->n_seqs) return fail(ctx, PA_EINVAL, "%s: sequence %u of %u", who, items[i].seq, L->n_seqs);
    if (items[i].pos >= 0x7fffffffu) return fail(ctx, PA_EINVAL, "%s: position %u is out of range", who, items[i].pos);
  }
  return PA_OK;
}

extern "C" int pa_decode_shared(pa_layer* L, pa_layer* prefix_layer, uint32_t prefix_seq, uint32_t prefix_len, uint32_t own_base, const pa_item* items,
                                uint32_t n_items, const void* q, int q_dtype, uint64_t qcs, uint64_t qhs, const void* gate, uint64_t gcs, uint64_t ghs, void* out,
                                uint64_t ocs, void* stream) {
  if (!L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  const char* who = "pa_decode_shared";
  if (int rc = shared_checks(L, items, n_items, q, q_dtype, out, who)) return rc;
  pa_layer* P = prefix_layer ? prefix_layer : L;
  const pa_ctx* pc = P->ctx;
  if (pc->failed) return fail(ctx, PA_ESTATE, "%s: an earlier step of the prefix layer's context failed (%s)", who, pc->err.c_str());
  if (P->kv_format != PA_KV_F16 || P->origin) return fail(ctx, PA_EUNSUPPORTED, "%s: the prefix must lie in an f16 cache that is no shard", who);
  if (pc->device != ctx->device || pc->cfg.n_kv_heads != ctx->cfg.n_kv_heads || pc->cfg.head_dim != ctx->cfg.head_dim)
    return fail(ctx, PA_EINVAL, "%s: the prefix layer is of another device or shape", who);
  if (prefix_seq >= P->n_seqs || prefix_len > P->max_seq)
    return fail(ctx, PA_EINVAL, "%s: rows [0, %u) of sequence %u: the prefix layer has %u sequences of %u rows", who, prefix_len, prefix_seq, P->n_seqs, P->max_seq);
  if (own_base && own_base != prefix_len) return fail(ctx, PA_EINVAL, "%s: own_base %u must be 0 or prefix_len %u", who, own_base, prefix_len);
  uint32_t rows[kMaxShared];
  for (uint32_t i = 0; i < n_items; ++i) {
    if (items[i].pos + 1 < prefix_len) return fail(ctx, PA_EINVAL, "%s: position %u lies inside the prefix of %u", who, items[i].pos, prefix_len);
    if (items[i].pos + 1 - own_base > L->max_seq) return fail(ctx, PA_EINVAL, "%s: position %u passes the layer's %u rows", who, items[i].pos, L->max_seq);
    rows[i] = items[i].pos + 1 - prefix_len;
  }
  SharedCall c{who, L, prefix_len ? P : nullptr, prefix_seq, prefix_len, prefix_len - own_base, q, q_dtype == PA_F16, qcs, qhs, gate, gcs, ghs, out, ocs, false};
  return shared_impl(c, items, n_items, rows, (cudaStream_t)stream);
}

extern "C" int pa_layer_track_weights(pa_layer* L) {
  if (!L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  if (L->kv_format != PA_KV_F16) return fail(ctx, PA_EUNSUPPORTED, "pa_layer_track_weights: f16 caches only");
  if (L->sums) return PA_OK;
  DeviceScope on(ctx->device);
  const size_t sums = (size_t)L->n_seqs * ctx->cfg.n_kv_heads * L->max_seq;
  // scores: a token of every sequence, up to 2^28 of them; never less than one item wants, nor than an eviction's lists
  const size_t one = scores_of(ctx, L->max_seq), want = std::max(std::max(one, sums), std::min<size_t>(one * L->n_seqs, (size_t)1 << 28));
  float *s = nullptr, *w = nullptr;
  try { ctx->outgrown.reserve(ctx->outgrown.size() + 1); } catch (...) { return fail(ctx, PA_ENOMEM, "pa_layer_track_weights: out of host memory"); }
  cudaError_t e = cudaMalloc(&s, sums * 4);
  if (e == cudaSuccess) e = cudaMemset(s, 0, sums * 4);
  if (e == cudaSuccess && want > ctx->scores_floats) e = cudaMalloc(&w, want * 4);
  if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
  if (e != cudaSuccess) {
    cudaGetLastError();
    cudaFree(s); cudaFree(w);
    return fail(ctx, e == cudaErrorMemoryAllocation ? PA_ENOMEM : PA_ECUDA, "pa_layer_track_weights: %.0f MiB of sums and %.0f MiB of scores: %s", sums * 4 / 1048576.0,
                want * 4 / 1048576.0, cudaGetErrorString(e));
  }
  L->sums = s;
  if (w) {
    if (ctx->scores) ctx->outgrown.push_back(ctx->scores);
    ctx->scores = w; ctx->scores_floats = want;
  }
  return PA_OK;
}
extern "C" float* pa_weights_ptr(pa_layer* L) { return L ? L->sums : nullptr; }

extern "C" int pa_weights_clear(pa_layer* L, uint32_t seq, void* stream) {
  if (!L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  if (!L->sums) return fail(ctx, PA_EINVAL, "pa_weights_clear: call pa_layer_track_weights first");
  if (seq >= L->n_seqs) return fail(ctx, PA_EINVAL, "pa_weights_clear: sequence %u of %u", seq, L->n_seqs);
  const size_t n = (size_t)ctx->cfg.n_kv_heads * L->max_seq;
  DeviceScope on(ctx->device);
  CU_TRY(ctx, cudaMemsetAsync(L->sums + seq * n, 0, n * 4, (cudaStream_t)stream));
  return PA_OK;
}

extern "C" int pa_decode_weights(pa_layer* L, const pa_item* items, uint32_t n_items, const void* q, int q_dtype, uint64_t qcs, uint64_t qhs, const void* gate,
                                 uint64_t gcs, uint64_t ghs, void* out, uint64_t ocs, void* stream) {
  if (!L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  const char* who = "pa_decode_weights";
  if (int rc = shared_checks(L, items, n_items, q, q_dtype, out, who)) return rc;
  if (!L->sums) return fail(ctx, PA_EINVAL, "%s: call pa_layer_track_weights first", who);
  uint32_t rows[kMaxShared];
  for (uint32_t i = 0; i < n_items; ++i) {
    if (items[i].pos >= L->max_seq) return fail(ctx, PA_EINVAL, "%s: position %u passes the layer's %u rows", who, items[i].pos, L->max_seq);
    rows[i] = items[i].pos + 1;
  }
  SharedCall c{who, L, nullptr, 0, 0, 0, q, q_dtype == PA_F16, qcs, qhs, gate, gcs, ghs, out, ocs, true};
  return shared_impl(c, items, n_items, rows, (cudaStream_t)stream);
}

extern "C" int pa_evict(pa_layer* L, const pa_evict_item* items, uint32_t n_items, uint32_t n_keep, uint32_t n_first, uint32_t n_recent, uint32_t* kept, void* stream) {
  if (!L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  if (L->kv_format != PA_KV_F16) return fail(ctx, PA_EUNSUPPORTED, "pa_evict: f16 caches only");
  if (L->origin) return fail(ctx, PA_EUNSUPPORTED, "pa_evict: not on a shard of longer sequences");
  if (!L->sums) return fail(ctx, PA_EINVAL, "pa_evict: call pa_layer_track_weights first");
  if (!items || n_items < 1 || n_items > (uint32_t)kMaxEvict) return fail(ctx, PA_EINVAL, "pa_evict: 1 to %d items per call", kMaxEvict);
  if (n_keep < 1 || n_keep > L->max_seq || (uint64_t)n_first + n_recent > n_keep)
    return fail(ctx, PA_EINVAL, "pa_evict: n_keep %u must be 1 .. %u and hold the first %u and the last %u rows", n_keep, L->max_seq, n_first, n_recent);
  if ((uintptr_t)kept & 3) return fail(ctx, PA_EINVAL, "pa_evict: kept is not aligned to its type");
  EvictParams p{};
  p.n_items = n_items; p.n_kv = ctx->cfg.n_kv_heads; p.hd = ctx->cfg.head_dim; p.max_seq = L->max_seq; p.n_keep = n_keep; p.n_first = n_first; p.n_recent = n_recent;
  p.k = L->k; p.v = L->v; p.sums = L->sums;
  for (uint32_t i = 0; i < n_items; ++i) {
    const pa_evict_item& it = items[i];
    if (it.src_seq >= L->n_seqs || it.dst_seq >= L->n_seqs) return fail(ctx, PA_EINVAL, "pa_evict: sequence %u of %u", std::max(it.src_seq, it.dst_seq), L->n_seqs);
    if (it.n_rows > L->max_seq) return fail(ctx, PA_EINVAL, "pa_evict: %u rows pass the layer's %u", it.n_rows, L->max_seq);
    if (it.n_rows > kEvictKeys * 8) return fail(ctx, PA_EUNSUPPORTED, "pa_evict: %u rows, at most %u", it.n_rows, kEvictKeys * 8);
    for (uint32_t j = 0; j < i; ++j)
      if (items[j].dst_seq == it.dst_seq || items[j].src_seq == it.dst_seq || items[j].dst_seq == it.src_seq)
        return fail(ctx, PA_EINVAL, "pa_evict: the destination of item %u or %u is named by the other", j, i);
    p.src[i] = it.src_seq; p.dst[i] = it.dst_seq; p.rows[i] = it.n_rows;
  }
  p.list = kept;
  if (!kept) {
    if ((uint64_t)n_items * p.n_kv * n_keep > ctx->scores_floats)
      return fail(ctx, PA_EUNSUPPORTED, "pa_evict: the lists of %u items do not fit the context's room; pass `kept` or fewer items", n_items);
    p.list = reinterpret_cast<uint32_t*>(ctx->scores);
  }
  DeviceScope on(ctx->device);
  CU_TRY(ctx, launch_evict(p, (uint32_t)ctx->sm_count, ctx->device, (cudaStream_t)stream));
  ctx->stats.kernel_launches += 2; ctx->stats.calls++;
  // rows of any number may still be on the move: what follows on this layer fetches nothing ahead of its wait
  ctx->inflight_layer = L; ctx->inflight_row0 = 0;
  return PA_OK;
}
