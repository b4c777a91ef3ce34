// C entry point of the tree decode (include/pooled_attn.h): checks, the plan of the units, launches.
#include <math.h>

#include <algorithm>

#include "pa_host.cuh"
#include "pa_params.cuh"

namespace pa {
cudaError_t launch_tree(const TreeParams& p, bool wide, const CUtensorMap& k, const CUtensorMap& v, uint32_t hd, uint32_t n_kv, int dev, cudaStream_t st);
cudaError_t launch_tree_finish(const TreeFinishParams& p, uint32_t hd, cudaStream_t st);
}  // namespace pa
using namespace pa;

static uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

// tiles of a run: f16 outputs at most 128, f32 at most 4 (10 with several row tiles; 24 where records run short), since the tensor cores'
// sums round towards zero.  (6 x 26 tokens of 24 / 4 heads of 256 behind up to 9001 rows: 55.5 us and off by 1.9e-6 of the largest output with runs of 16, 58 us
// and 1.2e-6 with 10; f32 products in the plain order 1.1e-6.)
static constexpr uint32_t kF16Tiles = 128, kF32Run = 24;
static uint32_t record_tiles(uint32_t T, uint32_t cap) { return ceil_div(T, ceil_div(T, cap)); }

// columns [first, first + cols) of an item
struct TreePart { uint32_t item, first, cols; };
struct TreePlan { uint32_t T; float us; };

// records of all rows with `T` tiles in each (parts in any order)
static uint64_t tree_records(const TreePart* parts, const uint32_t* tiles, uint32_t n, uint32_t n_heads, uint32_t T) {
  uint64_t sum = 0;
  for (uint32_t i = 0; i < n; ++i) sum += (uint64_t)parts[i].cols * n_heads * ceil_div(tiles[i], T);
  return sum;
}

// Tiles a unit (T), and the time that the launch takes with them: units one CTA an SM at a time (two of head_dim 128 and 64), the longest
// first, at the costs of a unit of T tiles, T * tile + start, and the records' way through L2.
static TreePlan plan_tree(const pa_ctx* ctx, const TreePart* parts, const uint32_t* tiles, const uint32_t* row_tiles, uint32_t n, bool wide, uint32_t tile_rows, uint32_t cap) {
  const uint32_t hd = ctx->cfg.head_dim, n_kv = ctx->cfg.n_kv_heads, sms = (uint32_t)ctx->sm_count * (hd == 256 ? 1 : 2);
  const float tile = hd == 256 ? (wide ? 1.22f : 0.77f) : wide ? 1.6f : 1.4f, start = wide ? 10.5f : 5.5f, record = 3.f * (float)tile_rows / 64;
  uint32_t longest = 1;
  float work_tiles = 0.f, hbm = 0.f;
  for (uint32_t i = 0; i < n; ++i) {
    longest = std::max(longest, tiles[i]);
    work_tiles += (float)(tiles[i] * row_tiles[i]);
    hbm += (float)tiles[i];
  }
  hbm *= (float)(n_kv * hd * 256) / 6.0e6f;
  TreePlan best{longest, 3.0e38f};
  for (uint32_t T = longest; T >= 1; T -= 1 + T / 40) {
    const uint32_t records = ceil_div(T, record_tiles(T, cap));
    uint32_t units = 0;
    uint64_t recs = 0;
    for (uint32_t i = 0; i < n; ++i) {
      const uint32_t splits = ceil_div(tiles[i], T);
      units += splits * row_tiles[i];
      recs += (uint64_t)parts[i].cols * splits;
    }
    units *= n_kv; recs *= ctx->cfg.n_heads;
    if (recs > ctx->tree_slots) break;
    const float unit = (float)T * tile + start + (float)(records - 1) * record;
    float us = units <= sms ? unit : std::max(unit, (work_tiles * n_kv * tile + (float)units * start) / (float)sms + 0.5f * unit);
    us = std::max(us, hbm + start) + (float)(recs * records * hd * 4) / 5.0e6f;
    if (us < best.us) best = TreePlan{T, us};
  }
  return best;
}

struct TreeCall {
  pa_layer* L;
  const pa_item* items;
  const uint32_t* item_col0;
  const int32_t* parents;
  const void* q; int q_f16; uint64_t qcs, qhs;
  const void* gate; uint64_t gcs, ghs;
  void* out; uint64_t ocs;
};

// one launch of each kernel for these parts, whose columns follow one another from `first_col` on
static int tree_launch(const TreeCall& c, const TreePart* parts, uint32_t n, uint32_t first_col, uint32_t cols, cudaStream_t st) {
  pa_layer* L = c.L;
  pa_ctx* ctx = L->ctx;
  const uint32_t hd = ctx->cfg.head_dim, nH = ctx->cfg.n_heads, n_kv = ctx->cfg.n_kv_heads, G = ctx->G;
  const size_t aes = ctx->cfg.act_dtype == PA_F16 ? 2 : 4;
  TreeParams p{};
  TreeFinishParams f{};
  uint32_t tiles[kMaxTrees], row_tiles[kMaxTrees], wide_tiles[kMaxTrees], most_row_tiles = 0, rows_of_tile = 0, total = 0;
  for (uint32_t i = 0; i < n; ++i) {
    tiles[i] = ceil_div(c.items[parts[i].item].pos + parts[i].first + parts[i].cols, 64);
    row_tiles[i] = ceil_div(parts[i].cols, 64 / G);
    wide_tiles[i] = ceil_div(parts[i].cols, 128 / G);
    most_row_tiles = std::max(most_row_tiles, row_tiles[i]);
    rows_of_tile = std::max(rows_of_tile, std::min(parts[i].cols, 64 / G) * G);
    f.col0[i] = total;
    total += parts[i].cols;
  }
  f.col0[n] = total;
  const bool f16_out = ctx->cfg.act_dtype == PA_F16;
  const uint32_t cap = f16_out ? kF16Tiles : most_row_tiles > 1 ? 10u : 4u;
  TreePlan plan = plan_tree(ctx, parts, tiles, row_tiles, n, false, rows_of_tile, cap);
  bool wide = false;
  if (most_row_tiles > 1 && c.q_f16 && f16_out && ctx->tune.shared_wide != 0) {
    const TreePlan w = plan_tree(ctx, parts, tiles, wide_tiles, n, true, 128, cap);
    if (w.us < plan.us || ctx->tune.shared_wide == 1) { plan = w; wide = true; }
  }
  // tiles of a record: a unit's shared out evenly; more where there is no room for that many, and past the
  // longest run a record adds up several
  uint32_t T = plan.T, records = ceil_div(T, cap);
  while (records > 1 && tree_records(parts, tiles, n, nH, ceil_div(T, records)) > ctx->tree_slots) --records;
  uint32_t rec = ceil_div(T, records);
  p.fold = ceil_div(rec, std::max(cap, kF32Run));
  rec = ceil_div(rec, p.fold) * p.fold;
  T = records * rec;
  p.seg = rec / p.fold; p.tps = T;
  // the longest first
  uint32_t order[kMaxTrees], recs = 0;
  for (uint32_t i = 0; i < n; ++i) {
    uint32_t j = i;
    for (; j && tiles[order[j - 1]] < tiles[i]; --j) order[j] = order[j - 1];
    order[j] = i;
    f.rec0[i] = recs; f.n_rec[i] = (uint16_t)ceil_div(tiles[i], rec);
    recs += parts[i].cols * nH * f.n_rec[i];
  }
  uint64_t read = 0;
  for (uint32_t k = 0; k < n; ++k) {
    const uint32_t i = order[k], rts = wide ? wide_tiles[i] : row_tiles[i];
    const pa_item& it = c.items[parts[i].item];
    p.seq[k] = it.seq; p.base[k] = it.pos; p.rows[k] = it.pos + parts[i].first + parts[i].cols;
    p.col0[k] = f.col0[i]; p.cols[k] = parts[i].cols; p.node0[k] = parts[i].first; p.parent0[k] = c.item_col0[parts[i].item];
    p.rec0[k] = f.rec0[i]; p.n_rec[k] = f.n_rec[i];
    p.tile_cols[k] = (uint16_t)ceil_div(parts[i].cols, rts);      // (evenly)
    p.row_tiles[k] = (uint16_t)ceil_div(parts[i].cols, p.tile_cols[k]);
    p.unit0[k] = p.units;
    p.units += ceil_div(tiles[i], T) * p.row_tiles[k];
    read += p.rows[k];
  }
  p.unit0[n] = p.units;
  p.q = reinterpret_cast<const uint8_t*>(c.q) + (uint64_t)first_col * c.qcs * (c.q_f16 ? 2 : 4); p.q_f16 = c.q_f16; p.q_col_stride = c.qcs; p.q_head_stride = c.qhs;
  p.n_heads = nH; p.G = G; p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
  p.part_o = ctx->part_o; p.part_ml = ctx->part_ml;
  p.parents = c.parents; p.v = L->v; p.kv_dim = ctx->kv_dim; p.max_seq = L->max_seq; p.n_items = n; p.err = ctx->dev_err;
  f.part_o = p.part_o; f.part_ml = p.part_ml; f.n_items = n; f.n_heads = nH; f.n_rows = cols * nH;
  f.gate = c.gate ? reinterpret_cast<const uint8_t*>(c.gate) + (uint64_t)first_col * c.gcs * aes : nullptr; f.gate_col_stride = c.gcs; f.gate_head_stride = c.ghs;
  f.out = reinterpret_cast<uint8_t*>(c.out) + (uint64_t)first_col * c.ocs * aes; f.out_col_stride = c.ocs; f.act_f16 = f16_out;
  f.vec = !((uintptr_t)f.out % (4 * aes)) && c.ocs % 4 == 0 && (!c.gate || (!((uintptr_t)f.gate % (4 * aes)) && c.gcs % 4 == 0 && c.ghs % 4 == 0));
  // warps for pieces of rows where that gives every SM enough of them; else a CTA a row, or a 64-dim slice of one with many records
  f.lanes = f.n_rows >= 4 * (uint32_t)ctx->sm_count ? 0 : f.n_rows * 2 <= (uint32_t)ctx->sm_count * 4 && p.n_rec[0] > 16 ? 16 : hd / 4;
  CU_TRY(ctx, launch_tree(p, wide, L->tm_k64, L->tm_v64, hd, n_kv, ctx->device, st));
  CU_TRY(ctx, launch_tree_finish(f, hd, st));
  ctx->stats.kernel_launches += 2;
  ctx->stats.kv_bytes_streamed += read * ctx->kv_dim * 4;
  return PA_OK;
}

extern "C" int pa_decode_tree(pa_layer* L, const pa_item* items, uint32_t n_items, const int32_t* parents, const void* q, int q_dtype, uint64_t qcs, uint64_t qhs,
                              const void* gate, uint64_t gcs, uint64_t ghs, void* out, uint64_t ocs, void* stream) {
  if (!L) return PA_EINVAL;
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  const char* who = "pa_decode_tree";
  if (L->kv_format != PA_KV_F16) return fail(ctx, PA_EUNSUPPORTED, "%s: f16 caches only", who);
  if (L->origin) return fail(ctx, PA_EUNSUPPORTED, "%s: not on a shard of longer sequences", who);
  if (ctx->G > 64) return fail(ctx, PA_EUNSUPPORTED, "%s: more than 64 query heads per kv head", who);
  if ((size_t)ctx->cfg.n_heads * 2 > ctx->tree_slots) return fail(ctx, PA_EUNSUPPORTED, "%s: more than %zu query heads", who, ctx->tree_slots / 2);
  if (!items || !q || !out) return fail(ctx, PA_EINVAL, "%s: null items, q or out", who);
  if (q_dtype != PA_F32 && q_dtype != PA_F16) return fail(ctx, PA_EINVAL, "%s: unknown q dtype", who);
  if (n_items < 1 || n_items > (uint32_t)kMaxTrees) return fail(ctx, PA_EINVAL, "%s: 1 to %d items per call", who, kMaxTrees);
  uint32_t col0[kMaxTrees], total = 0;
  for (uint32_t i = 0; i < n_items; ++i) {
    const pa_item& it = items[i];
    if (it.seq >= L->n_seqs) return fail(ctx, PA_EINVAL, "%s: sequence %u of %u", who, it.seq, L->n_seqs);
    if (it.n_cols < 1 || it.n_cols > 256) return fail(ctx, PA_EINVAL, "%s: item %u has %u tokens, 1 to 256 are possible", who, i, it.n_cols);
    if ((uint64_t)it.pos + it.n_cols > L->max_seq)
      return fail(ctx, PA_EINVAL, "%s: item %u: %u tokens from row %u on pass the layer's %u rows", who, i, it.n_cols, it.pos, L->max_seq);
    col0[i] = total;
    total += it.n_cols;
  }
  const uint64_t am = q_dtype == PA_F16 ? 7 : 3;
  if ((qcs & am) || (qhs & am) || ((uintptr_t)q & 15)) return fail(ctx, PA_EINVAL, "%s: q strides must be multiples of 16 bytes and q 16-byte aligned", who);
  const uint32_t ae = ctx->cfg.act_dtype == PA_F16 ? 2 : 4;
  if ((uintptr_t)gate % ae || (uintptr_t)out % ae || ((uintptr_t)parents & 3)) return fail(ctx, PA_EINVAL, "%s: a pointer is not aligned to its type", who);
  if (total > 1 && ocs < ctx->q_dim) return fail(ctx, PA_EINVAL, "%s: the column stride of out is below %u", who, ctx->q_dim);
  const TreeCall c{L, items, col0, parents, q, q_dtype == PA_F16, qcs, qhs, gate, gcs, ghs, out, ocs};
  DeviceScope on(ctx->device);
  // columns that fit the records, two a row at least, go in one launch; a tree may be parted
  const uint32_t most = std::max<uint32_t>(1, (uint32_t)(ctx->tree_slots / (2 * (size_t)ctx->cfg.n_heads)));
  for (uint32_t col = 0, item = 0, in = 0; col < total;) {
    TreePart parts[kMaxTrees];
    uint32_t n = 0, cols = 0;
    while (item < n_items && cols < most) {
      const uint32_t take = std::min(items[item].n_cols - in, most - cols);
      parts[n++] = TreePart{item, in, take};
      cols += take; in += take;
      if (in == items[item].n_cols) { ++item; in = 0; }
    }
    if (int rc = tree_launch(c, parts, n, col, cols, (cudaStream_t)stream)) return rc;
    col += cols;
  }
  ctx->stats.calls++;
  ctx->inflight_layer = nullptr;         // these kernels wait for everything before them and write no cache row
  return PA_OK;
}
