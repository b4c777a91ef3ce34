// Rows of caches copied, forked and moved together (pa_cache_move): K, V, scales and summed weights of all items and layers in one
// launch.
//
// A tile is 2048 units (16 bytes of K or V, 4 bytes of scales and sums) of one item's rows in one array; a CTA loads it into
// registers, eight units a thread, and stores it.  Rows of a range lie one behind the other, so its tiles are runs of memory;
// tiles of listed rows are whole rows.  Items with the same source are one group whose tiles are loaded once and stored at each
// destination.
//
// Rows that move over one another (destination and source of an item overlap) may not be stored before they have been read:
//   up to 512 rows    a tile is a few columns of all the rows, and the CTA's barrier between loading and storing is enough: no
//                     order between tiles (the accepted paths of 8 trees in 8 layers of 8 x 128: 3.9 us)
//   more              tiles are taken in the rows' order (from the side that they move to; from a counter, since the order in which
//                     CTAs start is not defined), a tile's byte says that it has been loaded, and a CTA waits, with its own tile in
//                     registers and its own byte set, for the one or two earlier tiles that its stores would overwrite.  Whoever
//                     took a lower number has loaded that tile or is about to, without waiting for anybody ahead of its byte, so
//                     every wait ends; one that runs out of looks all the same leaves its tile unstored.  (The next number taken
//                     when the tile's loads are out: 70 us for 57, others wait for a tile whose CTA is still busy with the one
//                     before.)  The CTA that is done last clears the words.
// What bounds it: HBM, a row read and written once (a prompt of 8000 rows forked to seven sequences in two layers 43.5 us, 0.92 of the measured rate); rows over
// one another the wait for the other tile's byte on top of it (0.78 to 0.80 for a gap of 2000 rows, 0.55 for one of a row); a few rows the launch and two trips to memory, list and rows.
#include <string.h>

#include <algorithm>

#include "pa_host.cuh"
#include "pa_params.cuh"

namespace pa {

constexpr uint32_t kMvThreads = 256, kMvUnits = kMoveUnits / kMvThreads;

template <int BYTES> struct MvUnit;
template <> struct MvUnit<16> { using T = uint4; };
template <> struct MvUnit<4> { using T = uint32_t; };

__device__ __forceinline__ uint32_t mv_row(uint32_t i, uint32_t per, uint32_t inv) { return per == 1 ? i : __umulhi(i, inv); }   // i / per, i below 2^16

// the number of values below `v` among list[0 .. n), ascending; all threads of the CTA
__device__ __forceinline__ uint32_t mv_below(const uint32_t* list, uint32_t n, uint32_t v) {
  uint32_t a = 0, b = n;                               // the answer lies in [a, b]
  while (a < b) {
    const uint32_t step = (b - a + kMvThreads - 1) / kMvThreads, at = a + threadIdx.x * step;
    const uint32_t k = (uint32_t)__syncthreads_count(at < b && list[at] < v);      // the first k of the values looked at are below
    if (k == 0) { b = a; }
    else { const uint32_t na = a + (k - 1) * step + 1; b = min(b, a + k * step); a = min(na, b); }
  }
  return a;
}

// The tile has been loaded; waits until the one or two earlier tiles [lo, hi] that read what it will overwrite have been, too.  False, for all
// threads, where that took more than p.polls looks: the tile may not be stored then, rows that nobody has read yet would be lost.
__device__ __forceinline__ bool mv_in_order(const MoveParams& p, uint8_t* said, uint32_t tile, uint32_t lo, uint32_t hi) {
  bool late = false;
  if (threadIdx.x < 2 && lo + threadIdx.x <= hi && lo + threadIdx.x < tile) {
    uint32_t there = 0;
    for (uint32_t i = 0; i < p.polls && !there; ++i) {
      asm volatile("ld.relaxed.gpu.u8 %0, [%1];" : "=r"(there) : "l"(said + lo + threadIdx.x) : "memory");
      if (!there && i > 64) __nanosleep(32);
    }
    late = !there;
    if (late) atomicMax(p.err, (uint32_t)WAIT_MOVE);
  }
  return !__syncthreads_or(late);
}
// All threads have their part of the tile (the barrier takes a word made of all of it: a thread without its values does not get there), so
// the byte need not be ordered behind anything: whoever sees it overwrites what is in registers here.
__device__ __forceinline__ uint32_t mv_mix(const uint4& x) { return x.x ^ x.y ^ x.z ^ x.w; }
__device__ __forceinline__ uint32_t mv_mix(uint32_t x) { return x; }
template <typename T>
__device__ __forceinline__ void mv_say(uint8_t* said, uint32_t tile, const T (&x)[kMvUnits]) {
  uint32_t w = 0;
#pragma unroll
  for (uint32_t k = 0; k < kMvUnits; ++k) w ^= mv_mix(x[k]);
  const uint32_t any = __syncthreads_or(w == 1u) ? 3u : 1u;
  if (threadIdx.x == 0) asm volatile("st.relaxed.gpu.u8 [%0], %1;" ::"l"(said + tile), "r"(any) : "memory");
}

// the number of the CTA's next tile (thread 0): taken when this one waits for nothing any more, ahead of its stores
__device__ __forceinline__ uint32_t mv_next(const MoveParams& p) { return threadIdx.x == 0 ? atomicAdd(p.words, 1u) : 0; }

// an array of a layer, and the rows of its sequences
struct MvArray { uint8_t* start; uint64_t seq_rows; uint32_t per, inv; };
template <int BYTES> __device__ __forceinline__ typename MvUnit<BYTES>::T* mv_at(const MvArray& a, uint32_t seq, uint32_t row) {
  return reinterpret_cast<typename MvUnit<BYTES>::T*>(a.start + (seq * a.seq_rows + row) * ((uint64_t)a.per * BYTES));
}

// a tile of a range: a run of units, counted from the end where rows move up over one another
template <int BYTES, bool ORDER>
__device__ __forceinline__ uint32_t move_run(const MoveParams& p, uint32_t g, uint32_t tile, const MvArray& a, uint8_t* said) {
  using T = typename MvUnit<BYTES>::T;
  const uint64_t total = (uint64_t)p.n[g] * a.per, e0 = (uint64_t)tile * kMoveUnits;
  const uint32_t len = (uint32_t)min((uint64_t)kMoveUnits, total - e0), i0 = p.item0[g], i1 = p.item0[g + 1];
  const bool up = p.flags[g] & MOVE_UP;
  const uint64_t first = up ? total - e0 - len : e0;   // the tile's first unit
  const T* from = mv_at<BYTES>(a, p.seq[g], p.row[g]) + first + threadIdx.x;
  T x[kMvUnits] = {};
#pragma unroll
  for (uint32_t k = 0; k < kMvUnits; ++k)
    if (k * kMvThreads + threadIdx.x < len) x[k] = from[k * kMvThreads];
  bool store = true;
  if constexpr (ORDER) {                               // (ranges over one another that are no columns are always taken in order)
    if (p.flags[g] & MOVE_OVER) {
      mv_say(said, tile, x);
      const uint64_t gap = (uint64_t)(up ? p.dst_row[i0] - p.row[g] : p.row[g] - p.dst_row[i0]) * a.per, e1 = e0 + len;
      uint32_t lo = 1, hi = 0;
      if (e1 > gap) { lo = (uint32_t)((e0 > gap ? e0 - gap : 0) / kMoveUnits); hi = (uint32_t)((e1 - gap - 1) / kMoveUnits); }
      store = mv_in_order(p, said, tile, lo, hi);
    }
  }
  const uint32_t next = ORDER ? mv_next(p) : 0;
  if (!store) return next;
  for (uint32_t i = i0; i < i1; ++i) {
    T* to = mv_at<BYTES>(a, p.dst_seq[i], p.dst_row[i]) + first + threadIdx.x;
#pragma unroll
    for (uint32_t k = 0; k < kMvUnits; ++k)
      if (k * kMvThreads + threadIdx.x < len) to[k * kMvThreads] = x[k];
  }
  return next;
}

// a tile of whole rows, listed ones, or of a few columns of all of an item's rows
template <int BYTES, bool ORDER>
__device__ __forceinline__ uint32_t move_rows_of(const MoveParams& p, uint32_t g, uint32_t tile, const MvArray& a, uint8_t* said) {
  using T = typename MvUnit<BYTES>::T;
  const uint32_t tid = threadIdx.x, n = p.n[g], i0 = p.item0[g];
  const bool columns = p.flags[g] & MOVE_COLUMNS;
  const uint32_t* list = p.lists ? p.lists + (uint64_t)p.list[i0] * p.list_stride : nullptr;
  const uint32_t most = list ? min(n, p.list_stride - 1) : n, rows = list ? min(list[0], most) : n;      // rows that may move, and that do
  uint32_t width = a.per, c0 = 0, first_row = 0, r_tile = kMoveUnits / a.per;
  if (columns) {
    r_tile = 1;
    while (r_tile < most) r_tile <<= 1;                // (the launcher's rule)
    width = min(a.per, kMoveUnits / r_tile); c0 = tile * width;
  } else {
    first_row = tile * r_tile;
  }
  const uint32_t live_rows = rows > first_row ? min(rows - first_row, r_tile) : 0, w_inv = width < a.per ? 2u << __clz(width) : a.inv;      // (columns: four at least, a power of two)
  const T* from = mv_at<BYTES>(a, p.seq[g], p.row[g]);
  T x[kMvUnits] = {};
  uint32_t to_at[kMvUnits];                            // units from the tile's first row at the destination; ~0: none
#pragma unroll
  for (uint32_t k = 0; k < kMvUnits; ++k) {
    const uint32_t r = mv_row(k * kMvThreads + tid, width, w_inv);
    to_at[k] = r < live_rows ? (list ? list[1 + first_row + r] : first_row + r) : n;      // the source row for now
  }
#pragma unroll
  for (uint32_t k = 0; k < kMvUnits; ++k) {
    const uint32_t i = k * kMvThreads + tid, r = mv_row(i, width, w_inv), c = c0 + i - r * width, src = to_at[k];
    const bool live = src < n && c < a.per;            // (a listed row past the item's: not moved)
    to_at[k] = live ? r * a.per + c : ~0u;
    if (live) x[k] = from[(uint64_t)src * a.per + c];
  }
  bool store = true;
  if (columns) {
    __syncthreads();                                   // all of the item's rows are in registers
  } else if constexpr (ORDER) {
    if (p.flags[g] & MOVE_OVER) {
      mv_say(said, tile, x);
      uint32_t lo = 1, hi = 0;
      const uint32_t gap = p.row[g] - p.dst_row[i0], past = first_row + live_rows;        // row r of the destination is row r - gap of the source
      if (live_rows && past > gap) {
        const uint32_t below = mv_below(list + 1, rows, first_row > gap ? first_row - gap : 0);
        lo = below / r_tile; hi = (below + live_rows - 1) / r_tile;
      }
      store = mv_in_order(p, said, tile, lo, hi);
    }
  }
  const uint32_t next = ORDER ? mv_next(p) : 0;
  if (!store) return next;
  T* to = mv_at<BYTES>(a, p.dst_seq[i0], p.dst_row[i0]) + (uint64_t)first_row * a.per;
#pragma unroll
  for (uint32_t k = 0; k < kMvUnits; ++k)
    if (to_at[k] != ~0u) to[to_at[k]] = x[k];
  return next;
}

template <bool ORDER, bool RUNS>
__device__ __forceinline__ uint32_t move_tile(const MoveParams& p, uint32_t unit) {
  // K and V of all layers, then their scales, then sums.  In order: the arrays of a kind take turns, so that a tile's neighbours in its own array
  // are further back (13937 rows of two sequences moved down by 2000, 4 x 256: 44 us for 56)
  uint32_t u = unit, kind = 0, arrays = 2 * p.n_layers;
  if (u >= arrays * p.tiles[0]) { u -= arrays * p.tiles[0]; kind = 1; }
  if (kind && u >= arrays * p.tiles[1]) { u -= arrays * p.tiles[1]; kind = 2; arrays = p.n_kv * p.n_layers; }
  const uint32_t v = ORDER ? u / arrays : u % p.tiles[kind], array = ORDER ? u - v * arrays : u / p.tiles[kind], of_layer = kind == 2 ? p.n_kv : 2, layer = array / of_layer, which = array - layer * of_layer;
  uint32_t g = 0, tile;
  if constexpr (ORDER && RUNS) {                       // ... and so do the groups: tile after tile of all that have that many
    uint32_t lo = 1, hi = p.n_groups;                  // m groups are left: at[m] <= v < at[m - 1]
    while (lo < hi) { const uint32_t mid = (lo + hi) / 2; if (p.at[kind][mid] <= v) hi = mid; else lo = mid + 1; }
    const uint32_t rest = v - p.at[kind][lo], c = lo < p.n_groups ? p.first[kind][lo + 1] - p.first[kind][lo] : 0;
    tile = c + rest / lo; g = rest % lo;
  } else {
    uint32_t hi = p.n_groups - 1;
    while (g < hi) { const uint32_t mid = (g + hi + 1) / 2; if (v >= p.first[kind][mid]) g = mid; else hi = mid - 1; }
    tile = v - p.first[kind][g];
  }
  uint8_t* said = ORDER ? reinterpret_cast<uint8_t*>(p.words + kMoveHead) + (unit - u) + array * p.tiles[kind] + p.first[kind][g] : nullptr;      // bytes of the group's tiles of this array
  MvArray a;
  if (kind == 0) a = MvArray{reinterpret_cast<uint8_t*>(p.rows[layer][which]), p.max_seq, p.per[0], p.inv[0]};
  else if (kind == 1) a = MvArray{reinterpret_cast<uint8_t*>(p.scales[layer][which]), p.max_seq, p.per[1], p.inv[1]};
  else a = MvArray{reinterpret_cast<uint8_t*>(p.sums[layer] ? p.sums[layer] + (uint64_t)which * p.max_seq : nullptr), (uint64_t)p.n_kv * p.max_seq, 1, 0};
  const bool run = RUNS || (!p.lists && !(p.flags[g] & MOVE_COLUMNS));
  if (kind == 0) {
    if (run) return move_run<16, ORDER>(p, g, tile, a, said);
    if constexpr (!RUNS) return move_rows_of<16, ORDER>(p, g, tile, a, said);
  } else if (a.start) {
    if (run) return move_run<4, ORDER>(p, g, tile, a, said);
    if constexpr (!RUNS) return move_rows_of<4, ORDER>(p, g, tile, a, said);
  }
  return ORDER ? mv_next(p) : 0;
}

// ORDER: CTAs that stay take tile after tile in their order; else a CTA a tile.  RUNS: no
// lists, no columns
constexpr int mv_ctas(bool runs) { return runs ? 5 : 4; }
template <bool ORDER, bool RUNS>
__global__ void __launch_bounds__(kMvThreads, mv_ctas(RUNS)) pa_move_kernel(const __grid_constant__ MoveParams p) {
  pdl_wait();
  pdl_trigger();
  if constexpr (!ORDER) {
    move_tile<false, RUNS>(p, blockIdx.x);
  } else {
    __shared__ uint32_t s_unit[2], s_done;
    if (threadIdx.x == 0) s_unit[0] = atomicAdd(p.words, 1u);
    __syncthreads();
    for (uint32_t i = 0;; ++i) {
      const uint32_t unit = s_unit[i & 1];
      if (unit >= p.units) break;
      const uint32_t next = move_tile<true, RUNS>(p, unit);
      if (threadIdx.x == 0) s_unit[(i + 1) & 1] = next;
      __syncthreads();
    }
    if (threadIdx.x == 0) { __threadfence(); s_done = atomicAdd(p.words + 1, 1u); }
    __syncthreads();
    if (s_done == gridDim.x - 1) {                     // nobody waits any more: the words are zero again for the next call
      __threadfence();
      uint32_t* w = p.words;
      for (uint32_t i = threadIdx.x; i < kMoveHead + (p.units + 3) / 4; i += kMvThreads) w[i] = 0;
    }
  }
}

}  // namespace pa
using namespace pa;

extern "C" int pa_cache_move(pa_layer* const* layers, uint32_t n_layers, const pa_move_item* items, uint32_t n_items, const uint32_t* lists, uint32_t list_stride,
                             void* stream) {
  if (!layers || n_layers < 1 || !layers[0]) return PA_EINVAL;
  pa_layer* L = layers[0];
  pa_ctx* ctx = L->ctx;
  GUARD(ctx);
  for (uint32_t i = 0; i < n_layers; ++i) {
    const pa_layer* l = layers[i];
    if (!l || l->ctx != ctx) return fail(ctx, PA_EINVAL, "pa_cache_move: layer %u of the call is null or of another context", i);
    if (l->kv_format != L->kv_format || l->n_seqs != L->n_seqs || l->max_seq != L->max_seq)
      return fail(ctx, PA_EINVAL, "pa_cache_move: layers of one call have one cache format and as many sequences and rows");
    for (uint32_t j = 0; j < i; ++j)
      if (layers[j] == l) return fail(ctx, PA_EINVAL, "pa_cache_move: layer %u of the call is layer %u again", i, j);
  }
  if (!items || n_items < 1 || n_items > (uint32_t)kMaxMoves) return fail(ctx, PA_EINVAL, "pa_cache_move: 1 to %d items per call", kMaxMoves);
  if (lists && (list_stride < 1 || ((uintptr_t)lists & 3))) return fail(ctx, PA_EINVAL, "pa_cache_move: lists are aligned words, one at least of each");
  const uint32_t es = L->kv_format == PA_KV_Q8 ? 1 : L->kv_format == PA_KV_F32 ? 4 : 2;
  MoveParams p{};
  p.per[0] = ctx->kv_dim * es / 16; p.per[1] = L->kv_format == PA_KV_Q8 ? ctx->kv_dim / 32 : 0;
  for (int k = 0; k < 2; ++k) p.inv[k] = p.per[k] > 1 ? (uint32_t)((0x100000000ull + p.per[k] - 1) / p.per[k]) : 0;
  if (lists && p.per[0] > kMoveUnits) return fail(ctx, PA_EUNSUPPORTED, "pa_cache_move: listed rows of at most %u bytes", kMoveUnits * 16);
  p.max_seq = L->max_seq; p.n_kv = ctx->cfg.n_kv_heads; p.lists = lists; p.list_stride = list_stride; p.err = ctx->dev_err;
  p.polls = ctx->tune.wait_polls ? ctx->tune.wait_polls : kMergePolls;
  bool sums = false;
  for (uint32_t i = 0; i < n_layers; ++i) sums = sums || layers[i]->sums;
  // which rows an item may read and write (a span without rows meets none)
  struct Span { uint32_t seq, a, b; };
  auto meet = [](const Span& x, const Span& y) { return x.seq == y.seq && std::max(x.a, y.a) < std::min(x.b, y.b); };
  Span from[kMaxMoves], to[kMaxMoves];
  for (uint32_t i = 0; i < n_items; ++i) {
    const pa_move_item& it = items[i];
    const uint32_t most = lists ? std::min(it.n_rows, list_stride - 1) : it.n_rows;
    if (it.src_seq >= L->n_seqs || it.dst_seq >= L->n_seqs) return fail(ctx, PA_EINVAL, "pa_cache_move: sequence %u of %u", std::max(it.src_seq, it.dst_seq), L->n_seqs);
    if ((uint64_t)it.src_row + it.n_rows > L->max_seq || (uint64_t)it.dst_row + most > L->max_seq)
      return fail(ctx, PA_EINVAL, "pa_cache_move: item %u: %u rows from row %u to row %u pass the layer's %u", i, it.n_rows, it.src_row, it.dst_row, L->max_seq);
    from[i] = Span{it.src_seq, it.src_row, it.src_row + it.n_rows};
    to[i] = Span{it.dst_seq, it.dst_row, it.dst_row + most};
    if (lists && meet(from[i], to[i]) && it.dst_row > it.src_row)
      return fail(ctx, PA_EINVAL, "pa_cache_move: item %u: listed rows do not move up over rows of their own item (row %u to row %u)", i, it.src_row, it.dst_row);
    for (uint32_t j = 0; j < i; ++j)
      if (meet(to[i], to[j]) || meet(to[i], from[j]) || meet(from[i], to[j]))
        return fail(ctx, PA_EINVAL, "pa_cache_move: items %u and %u: one stores rows that the other reads or stores", j, i);
  }
  // groups, and their tiles of each kind
  uint32_t total[3] = {0, 0, 0};
  bool order = false, runs = !lists, used[kMaxMoves] = {};
  uint32_t n = 0, by_rows[kMaxMoves];                  // items placed; the items, most rows first
  for (uint32_t i = 0; i < n_items; ++i) {
    uint32_t j = i;
    for (; j && items[by_rows[j - 1]].n_rows < items[i].n_rows; --j) by_rows[j] = by_rows[j - 1];
    by_rows[j] = i;
  }
  for (uint32_t b = 0; b < n_items; ++b) {
    const uint32_t i = by_rows[b];
    const pa_move_item& it = items[i];
    const uint32_t most = to[i].b - to[i].a;
    if (used[i] || !most || (!lists && it.src_seq == it.dst_seq && it.src_row == it.dst_row)) continue;
    const uint32_t g = p.n_groups++;
    const bool over = meet(from[i], to[i]), columns = over && most <= kMoveColumnRows;
    p.seq[g] = it.src_seq; p.row[g] = it.src_row; p.n[g] = it.n_rows; p.item0[g] = n;
    p.flags[g] = (over ? MOVE_OVER : 0) | (over && it.dst_row > it.src_row ? MOVE_UP : 0) | (columns ? MOVE_COLUMNS : 0);
    for (uint32_t j = i; j < n_items; ++j) {
      const pa_move_item& o = items[j];
      if (j > i && (over || lists || used[j] || o.src_seq != it.src_seq || o.src_row != it.src_row || o.n_rows != it.n_rows || (o.dst_seq == o.src_seq && o.dst_row == o.src_row))) continue;
      used[j] = true;
      p.dst_seq[n] = o.dst_seq; p.dst_row[n] = o.dst_row; p.list[n] = j;
      ++n;
    }
    order = order || (over && !columns);
    runs = runs && !columns;
    for (int k = 0; k < 3; ++k) {
      const uint32_t per = k == 2 ? 1 : p.per[k];
      p.first[k][g] = total[k];
      if (!per || (k == 2 && !sums)) continue;
      uint32_t r = 1;
      while (columns && r < most) r <<= 1;             // rows of a tile of columns, a power of two
      const uint64_t tiles = columns ? (per + std::min(per, kMoveUnits / r) - 1) / std::min(per, kMoveUnits / r)
                             : lists ? (most + kMoveUnits / per - 1) / (kMoveUnits / per) : ((uint64_t)most * per + kMoveUnits - 1) / kMoveUnits;
      if (total[k] + tiles > 0x10000000ull) return fail(ctx, PA_EUNSUPPORTED, "pa_cache_move: more rows than one call moves");
      total[k] += (uint32_t)tiles;
    }
  }
  ctx->stats.calls++;
  if (!p.n_groups) return PA_OK;
  p.item0[p.n_groups] = n;
  for (int k = 0; k < 3; ++k) {
    p.first[k][p.n_groups] = total[k]; p.tiles[k] = total[k];
    for (uint32_t m = p.n_groups; runs && m-- > 0;)    // (m + 1 groups take turns from the number of tiles of group m + 1 to that of group m)
      p.at[k][m] = p.at[k][m + 1] + (m + 1) * (p.first[k][m + 1] - p.first[k][m] - (m + 1 < p.n_groups ? p.first[k][m + 2] - p.first[k][m + 1] : 0));
  }
  const uint64_t layer_tiles = 2ull * total[0] + 2ull * total[1] + (uint64_t)p.n_kv * total[2];
  const uint64_t most_layers = std::min<uint64_t>(kMoveLayers, (order ? (uint64_t)kMoveTiles : 0x7fffffffull) / layer_tiles);
  if (!most_layers) return fail(ctx, PA_EUNSUPPORTED, "pa_cache_move: %llu tiles of 32 KB of a layer, %u are moved over one another at most", (unsigned long long)layer_tiles, kMoveTiles);
  p.words = order ? ctx->move_words : nullptr;
  DeviceScope on(ctx->device);
  for (uint32_t l0 = 0; l0 < n_layers; l0 += (uint32_t)most_layers) {
    const uint32_t nl = std::min((uint32_t)most_layers, n_layers - l0);
    for (uint32_t i = 0; i < nl; ++i) {
      const pa_layer* l = layers[l0 + i];
      p.rows[i][0] = l->kv_format == PA_KV_F16 ? (void*)l->k : l->k_alt; p.rows[i][1] = l->kv_format == PA_KV_F16 ? (void*)l->v : l->v_alt;
      p.scales[i][0] = l->k_scale; p.scales[i][1] = l->v_scale; p.sums[i] = l->sums;
    }
    p.n_layers = nl; p.units = (uint32_t)(nl * layer_tiles);
    const dim3 grid(order ? std::min(p.units, (uint32_t)(ctx->sm_count * mv_ctas(runs))) : p.units);
    auto* kernel = order ? (runs ? pa_move_kernel<true, true> : pa_move_kernel<true, false>) : (runs ? pa_move_kernel<false, true> : pa_move_kernel<false, false>);
    CU_TRY(ctx, launch_pdl(kernel, grid, dim3(kMvThreads), 0, (cudaStream_t)stream, p));
    ctx->stats.kernel_launches++;
  }
  // rows of any number of these layers may still be on the move: what follows on them fetches nothing ahead of its wait
  ctx->inflight_layer = n_layers == 1 ? L : kEveryLayer; ctx->inflight_row0 = 0;
  return PA_OK;
}
