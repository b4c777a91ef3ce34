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
//                     order between tiles (the accepted paths of 8 trees in 8 layers of 8 x 128: 4.6 us a call)
//   more              tiles are taken in the rows' order (from the side that they move to; a counter, since the order in which CTAs
//                     start is not defined), a tile's byte says that it has been loaded, and a CTA waits, with its own tile in
//                     registers and its own byte set, for the one or two earlier tiles that its stores would overwrite.  A CTA
//                     with a lower number is running or done and sets its byte without waiting for anybody, so every wait ends.
//                     The CTA that is done last clears the words.
// What bounds it: HBM, a row read and written once (a prompt of 8000 rows forked to seven sequences in two layers 43 us, 0.92 of the measured rate); a few rows the launch and two trips to memory, list and rows.
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

// one tile of an array: `from` and `to` begin with the group's source row and, item by item, its destination row
template <int BYTES>
__device__ __forceinline__ void move_tile(const MoveParams& p, uint32_t g, uint32_t tile, uint32_t per, uint32_t inv, uint8_t* array, uint64_t seq_rows, bool ordered,
                                          uint8_t* said) {
  using T = typename MvUnit<BYTES>::T;
  const uint32_t tid = threadIdx.x, n = p.n[g], i0 = p.item0[g], i1 = p.item0[g + 1], flags = p.flags[g];
  const bool over = flags & MOVE_OVER, up = flags & MOVE_UP, columns = flags & MOVE_COLUMNS;
  const uint64_t row_bytes = (uint64_t)per * BYTES;
  auto at_row = [&](uint32_t seq, uint32_t row) { return reinterpret_cast<T*>(array + (seq * seq_rows + row) * row_bytes); };
  const T* from = at_row(p.seq[g], p.row[g]);
  const uint32_t* list = p.lists ? p.lists + (uint64_t)p.list[i0] * p.list_stride : nullptr;
  const uint32_t most = list ? min(n, p.list_stride - 1) : n, rows = list ? min(list[0], most) : n;      // rows that may move, and that do
  T x[kMvUnits];
  uint64_t to_at[kMvUnits];                            // units from the destination's start; ~0: none
  uint32_t first_row = 0, past_row = 0;                // of a tile of whole rows
  const uint64_t total = (uint64_t)rows * per;
  if (list || columns) {
    // whole rows, or `width` columns of all of them
    uint32_t width = per, c0 = 0, r_tile;
    if (columns) {
      r_tile = 1;
      while (r_tile < most) r_tile <<= 1;              // (the launcher's rule)
      width = min(per, kMoveUnits / r_tile); c0 = tile * width;
    } else {
      r_tile = kMoveUnits / per;
      first_row = tile * r_tile;
    }
    past_row = min(rows, first_row + r_tile);
    const uint32_t w_inv = width < per ? 2u << __clz(width) : inv;         // (columns: four at least, a power of two)
    uint32_t row[kMvUnits], src[kMvUnits];
#pragma unroll
    for (uint32_t k = 0; k < kMvUnits; ++k) {
      const uint32_t i = k * kMvThreads + tid, r = mv_row(i, width, w_inv);
      row[k] = first_row + r;
      src[k] = row[k] < past_row ? (list ? list[1 + row[k]] : row[k]) : n;
    }
#pragma unroll
    for (uint32_t k = 0; k < kMvUnits; ++k) {
      const uint32_t i = k * kMvThreads + tid, c = c0 + i - mv_row(i, width, w_inv) * width;
      const bool live = src[k] < n && c < per;         // (a listed row past the item's: not moved)
      to_at[k] = live ? (uint64_t)row[k] * per + c : ~0ull;
      if (live) x[k] = from[(uint64_t)src[k] * per + c];
    }
  } else {
#pragma unroll
    for (uint32_t k = 0; k < kMvUnits; ++k) {
      const uint64_t e = (uint64_t)tile * kMoveUnits + k * kMvThreads + tid;
      to_at[k] = e < total ? (up ? total - 1 - e : e) : ~0ull;
      if (e < total) x[k] = from[to_at[k]];
    }
  }
  if (over) {
    if (ordered) __threadfence();                      // this thread's loads are done
    __syncthreads();
    if (ordered) {
      if (tid == 0) asm volatile("st.release.gpu.u8 [%0], %1;" ::"l"(said + tile), "r"(1u) : "memory");
      // the tiles that read what this one overwrites
      uint32_t lo = 1, hi = 0;
      if (list) {
        const uint32_t gap = p.row[g] - p.dst_row[i0];                     // row r of the destination is row r - gap of the source
        if (past_row > gap && past_row > first_row) {
          const uint32_t r_tile = kMoveUnits / per, a = mv_below(list + 1, rows, first_row > gap ? first_row - gap : 0), b = a + (past_row - first_row);
          lo = a / r_tile; hi = (b - 1) / r_tile;
        }
      } else {
        const uint64_t gap = (uint64_t)(up ? p.dst_row[i0] - p.row[g] : p.row[g] - p.dst_row[i0]) * per, e0 = (uint64_t)tile * kMoveUnits,
                       e1 = min(total, e0 + kMoveUnits);
        if (e1 > gap && e1 > e0) { lo = (uint32_t)((e0 > gap ? e0 - gap : 0) / kMoveUnits); hi = (uint32_t)((e1 - gap - 1) / kMoveUnits); }
      }
      if (tid < 2 && lo + tid <= hi && lo + tid < tile) {
        uint32_t there = 0;
        for (uint32_t i = 0; i < kWaitPolls && !there; ++i) {
          asm volatile("ld.acquire.gpu.u8 %0, [%1];" : "=r"(there) : "l"(said + lo + tid) : "memory");
          if (!there && i > 64) __nanosleep(32);
        }
        if (!there) atomicMax(p.err, (uint32_t)WAIT_MOVE);
      }
      __syncthreads();
    }
  }
  for (uint32_t i = i0; i < i1; ++i) {
    T* to = at_row(p.dst_seq[i], p.dst_row[i]);
#pragma unroll
    for (uint32_t k = 0; k < kMvUnits; ++k)
      if (to_at[k] != ~0ull) to[to_at[k]] = x[k];
  }
}

template <bool ORDER>
__global__ void __launch_bounds__(kMvThreads) pa_move_kernel(const __grid_constant__ MoveParams p) {
  __shared__ uint32_t s_word;
  pdl_wait();
  pdl_trigger();
  uint32_t unit = blockIdx.x;
  if (ORDER) {
    if (threadIdx.x == 0) s_word = atomicAdd(p.words, 1u);
    __syncthreads();
    unit = s_word;
  }
  const uint32_t layer = unit / p.layer_tiles;
  uint32_t u = unit - layer * p.layer_tiles, kind = 0, which;
  if (u >= 2 * p.tiles[0]) { u -= 2 * p.tiles[0]; kind = 1; }
  if (kind && u >= 2 * p.tiles[1]) { u -= 2 * p.tiles[1]; kind = 2; }
  which = u / p.tiles[kind];
  u -= which * p.tiles[kind];
  uint32_t g = 0, hi = p.n_groups - 1;
  while (g < hi) { const uint32_t mid = (g + hi + 1) / 2; if (u >= p.first[kind][mid]) g = mid; else hi = mid - 1; }
  const uint32_t tile = u - p.first[kind][g];
  uint8_t* said = ORDER ? reinterpret_cast<uint8_t*>(p.words + kMoveHead) + (unit - tile) : nullptr;      // the bytes of the group's tiles of this array
  const bool ordered = ORDER && (p.flags[g] & (MOVE_OVER | MOVE_COLUMNS)) == MOVE_OVER;
  if (kind == 0) move_tile<16>(p, g, tile, p.per[0], p.inv[0], reinterpret_cast<uint8_t*>(p.rows[layer][which]), p.max_seq, ordered, said);
  else if (kind == 1) move_tile<4>(p, g, tile, p.per[1], p.inv[1], reinterpret_cast<uint8_t*>(p.scales[layer][which]), p.max_seq, ordered, said);
  else if (p.sums[layer])
    move_tile<4>(p, g, tile, 1, 0, reinterpret_cast<uint8_t*>(p.sums[layer] + (uint64_t)which * p.max_seq), (uint64_t)p.n_kv * p.max_seq, ordered, said);
  if (ORDER) {
    __syncthreads();
    if (threadIdx.x == 0) { __threadfence(); s_word = atomicAdd(p.words + 1, 1u); }
    __syncthreads();
    if (s_word == gridDim.x - 1) {                     // everybody is done: the words are zero again for the next call
      __threadfence();
      uint32_t* w = p.words;
      for (uint32_t i = threadIdx.x; i < kMoveHead + (gridDim.x + 3) / 4; i += kMvThreads) w[i] = 0;
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
  bool sums = false;
  for (uint32_t i = 0; i < n_layers; ++i) sums = sums || layers[i]->sums;
  // which rows an item may read and write
  struct Span { uint32_t seq, a, b; };
  auto meet = [](const Span& x, const Span& y) { return x.seq == y.seq && x.a < y.b && y.a < x.b; };
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
  bool order = false, used[kMaxMoves] = {};
  uint32_t n = 0;                                      // items placed
  for (uint32_t i = 0; i < n_items; ++i) {
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
  for (int k = 0; k < 3; ++k) { p.first[k][p.n_groups] = total[k]; p.tiles[k] = total[k]; }
  const uint64_t layer_tiles = 2ull * total[0] + 2ull * total[1] + (uint64_t)p.n_kv * total[2];
  const uint64_t most_layers = std::min<uint64_t>(kMoveLayers, (order ? (uint64_t)kMoveTiles : 0x7fffffffull) / layer_tiles);
  if (!most_layers) return fail(ctx, PA_EUNSUPPORTED, "pa_cache_move: %llu tiles of 32 KB of a layer, %u are moved over one another at most", (unsigned long long)layer_tiles, kMoveTiles);
  p.layer_tiles = (uint32_t)layer_tiles;
  p.words = order ? ctx->move_words : nullptr;
  DeviceScope on(ctx->device);
  for (uint32_t l0 = 0; l0 < n_layers; l0 += (uint32_t)most_layers) {
    const uint32_t nl = std::min((uint32_t)most_layers, n_layers - l0);
    for (uint32_t i = 0; i < nl; ++i) {
      const pa_layer* l = layers[l0 + i];
      p.rows[i][0] = l->kv_format == PA_KV_F16 ? (void*)l->k : l->k_alt; p.rows[i][1] = l->kv_format == PA_KV_F16 ? (void*)l->v : l->v_alt;
      p.scales[i][0] = l->k_scale; p.scales[i][1] = l->v_scale; p.sums[i] = l->sums;
    }
    const dim3 grid((uint32_t)(nl * layer_tiles));
    CU_TRY(ctx, order ? launch_pdl(pa_move_kernel<true>, grid, dim3(kMvThreads), 0, (cudaStream_t)stream, p) : launch_pdl(pa_move_kernel<false>, grid, dim3(kMvThreads), 0, (cudaStream_t)stream, p));
    ctx->stats.kernel_launches++;
  }
  // rows of any number of these layers may still be on the move: what follows on them fetches nothing ahead of its wait
  ctx->inflight_layer = n_layers == 1 ? L : kEveryLayer; ctx->inflight_row0 = 0;
  return PA_OK;
}
