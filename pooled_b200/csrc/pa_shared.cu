// Attention of a batch of single tokens that share their first rows (pa_decode_shared), and of a batch whose weights are summed
// per cached row (pa_decode_weights): one kernel over both kinds of rows, and one that merges.
//
//   o = sum_r e^(q.k_r / sqrt(hd) - M) v_r / sum_r e^(q.k_r / sqrt(hd) - M)   over the shared rows and the item's own
//
// A unit is a run of 64-row K / V tiles of one kv head and the query rows that attend them: for the shared rows the heads of
// several items (so that a shared byte is read once for all of these, from HBM once in all), for own rows the heads of one.
// A CTA per unit walks its tiles on the 5th-generation tensor cores and leaves an unnormalised (o, m, l) record per query
// row, or one for every p.seg tiles: the tensor cores' sums round towards zero, which after 32 tiles has cost 2.3e-6 of the result, after
// four 6e-7, after 2344 1.5e-4, so with f32 outputs a run has at most 4 tiles (16 where the tensor cores bound the call, 24 where there is no room
// for that many records), with f16 ones 128; longer records are the f32 sum of p.fold runs.  The second
// kernel merges a row's records, gates and stores.  All units have the same number
// of tiles, whatever they are units of (plan_units), so that a batch of long shared rows and short own ones fills the machine
// like one long conversation.
//
//   warps 0, 3  TMA producers: K tiles and V tiles (64 x head_dim f16, 128-byte swizzle), a ring of three and of two slots;
//               warp 3 then clears the rows of the last V tile that lie behind the unit's last: a weight of zero does not
//               make up for an infinity or NaN that the cache holds there
//   warp 1      issues the scores: S = Q K^T into one of two or three tiles of tensor memory (128 x 64 f32)
//   warp 2      tensor memory; issues O += P V into the accumulator (128 x head_dim f32)
//   warps 4-11  softmax, two groups of four warps with half of a tile's keys each (on alternate tiles, a call of one tile a CTA took
//               0.4 us longer, and wide tiles 1.5 us each).  A row's reference lies 2^7 below its maximum and moves only when a tile
//               passes it by 2^15: weights of up to 2^15 keep the low parts of small ones above f16's last place.  Warps whose rows
//               hold no query take no part
// q and the weights enter as pairs of f16 values, high and low parts, some 22 bits of both, in one of two ways:
//   narrow (up to 64 query rows)   even rows of the 128 carry the high parts, odd rows the low parts of the same query row, added by
//               shuffles: both products at the cost of one, and the two lanes share the row's keys out.  0.75 us a tile of 64 keys
//               at head_dim 256 (the tensor cores: 1394 cycles); 0.67 at 128 and 64 (the chain through the softmax), 0.8 of two
//               CTAs an SM
//   wide (head_dim 256, f16 queries and outputs, shared rows of more than 64 query rows, where the plan finds it faster)   128 query
//               rows without low parts of q; the low parts of the weights are multiplied behind the high ones into the same
//               accumulator.  1.17 us a tile and a start 5 us longer: 32 items of 8 heads behind 32768 rows 35 us, narrow 39, and
//               32 with weights of one f16 value, whose rounding would add as much error as the output's own.  (With f32
//               queries and the products of their low parts 1.43 us and 13 us of start, slower than two narrow tiles at every size
//               tried; at head_dim 128 0.64 us, slower than two narrow CTAs an SM.)
// What bounds it: HBM, one query tile per kv head and long rows; several, the tensor cores within a unit (33 % of a launch at 32 items: the
// rest is starts, ends and records); short calls the chain of launch, q,
// scores, weights, products and records, and fetching the code for it: without wide units a kernel of half the code runs.
#include "pa_shared.cuh"

namespace pa {

// grid (kv heads, units): the shared rows' units of all heads first.  MIXED: they are wide (an instantiation of its own: calls without wide
// units run a kernel of half the code, most of whose time at short rows is fetching it).  FOLD: records of several runs, wide units of several (likewise: as a
// branch it made calls that have none 0.1 to 0.3 us slower)
template <int HD, bool MIXED, bool FOLD>
__global__ void __launch_bounds__(384, ShSmem<HD>::CTAS)
pa_shared_kernel(const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ SharedParams p) {
  using L = ShSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::OFF_BAR);
  volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(bars + 31);
  volatile uint32_t* s_err = s_tmem + 1;
  const uint32_t bar0 = smem_u32(bars);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t unit = blockIdx.y;
  ShUnit un;
  un.shared = unit < p.p_splits * p.row_tiles;
  uint32_t split, n_q, tps;
  if (un.shared) {
    split = unit / p.row_tiles;
    un.item0 = (unit % p.row_tiles) * p.items_per_tile;
    n_q = min(p.items_per_tile, p.n_items - un.item0);
    un.row0 = p.p_row0; un.n_rows = p.p_rows; tps = p.p_tps; un.slot = 0;
    un.mk = &tm_pk; un.mv = &tm_pv;
  } else {
    uint32_t lo = 0, hi = p.n_items - 1;
    while (lo < hi) { const uint32_t mid = (lo + hi + 1) / 2; if (unit >= p.cta0[mid]) lo = mid; else hi = mid - 1; }
    un.item0 = lo; n_q = 1; split = unit - p.cta0[lo];
    un.row0 = p.seq[lo] * p.max_seq + p.own_row0; un.n_rows = p.rows[lo]; tps = p.tps; un.slot = p.p_recs;
    un.mk = &tm_k; un.mv = &tm_v;
  }
  un.tile0 = split * tps;
  un.slot += un.tile0 / (FOLD ? p.seg * p.fold : p.seg);                // (tiles per unit: a multiple of a record's)
  un.n_tiles = min((un.n_rows + 63) / 64, un.tile0 + tps) - un.tile0;
  un.pairs = n_q * p.G;
  const bool wide = MIXED && un.shared;
  un.live_warps = ((wide ? 1 : 2) * un.pairs + 31) / 32;
  un.ragged = (un.tile0 + un.n_tiles) * 64 > un.n_rows;

  if (warp == 1 && lane == 0) {
    *s_err = 0;
    auto init = [&](int which, int n, uint32_t count) { for (int i = 0; i < n; ++i) mbar_init(bar0 + 8u * (uint32_t)(which + i), count); };
    init(SH_K_FULL, 3, 1); init(SH_K_EMPTY, 3, 1); init(SH_V_FULL, 2, 1); init(SH_V_EMPTY, 2, 1);
    init(SH_S_FULL, 3, 1); init(SH_P_FULL, 3, 64 * un.live_warps); init(SH_PV_DONE, 3, 1);
    init(SH_O_DONE, 1, 1); init(SH_O_FREE, 1, 64 * un.live_warps); init(SH_Q_FULL, 1, 256); init(SH_Q_READ, 1, 256); init(SH_V_CLEAN, 1, 1);
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(smem_u32((const void*)s_tmem), sh_tmem_cols<HD>());
    tmem_relinquish();
    tc_fence_before();
  }
  if (warp == 0 && lane == 0) { prefetch_tmap(un.mk); prefetch_tmap(un.mv); }
  pdl_wait();
  pdl_trigger();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  if (warp == 0 || warp == 3) {
    shared_producer<HD>(un, warp == 3, base, bar0, s_err);
  } else {
    if constexpr (MIXED) {
      if (wide) shared_roles<HD, true, false, FOLD>(p, un, base, bar0, s_err, tmem);
    }
    if (!wide) shared_roles<HD, false, !MIXED, FOLD>(p, un, base, bar0, s_err, tmem);
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, sh_tmem_cols<HD>());
  }
  if (tid == 0 && *s_err) atomicMax(p.err, *s_err);
}

// ------------------------------------------------------------------------------ merge and sums --

// CTAs below merge_ctas merge: one (item, head) each, or one 64-dim slice of it where there are many records and few rows to
// share them out (p.lanes: float4 lanes of a CTA's part of the row).  Every warp finds the row's maximum and sum by itself, over
// records requested together with the (m, l) pairs, so that nothing waits for a barrier but the sum of the groups of lanes.
// The others: kSumRows rows of a sequence and kv head; the final (m, l) of the group's heads from their records while the
// scores are on their way, then per row sum_h 2^(s_h - m_h) / l_h, added to the row's sum: four threads a row, each with
// every fourth head, then the four in order, item after item.
template <int HD, bool SUMS>
__global__ void __launch_bounds__(256, SUMS ? 3 : 4) pa_shared_finish_kernel(const __grid_constant__ SharedFinishParams p) {
  __shared__ float4 s_acc[256];
  __shared__ float s_m[64], s_il[64];
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  if (!SUMS || blockIdx.x < p.merge_ctas) {
    const uint32_t slices = HD / 4 / p.lanes, prow = blockIdx.x / slices, slice = blockIdx.x % slices, item = prow / p.n_heads, h = prow % p.n_heads;
    shared_merge_row<HD>(p, s_acc, (uint64_t)prow * p.n_rec, slice, item, h, p.p_recs + p.n_own[item]);
    return;
  }
  if constexpr (SUMS) {
    // ---- sums of the weights ----
    const uint32_t u0 = blockIdx.x - p.merge_ctas;
    uint32_t lo = 0, hi = p.n_leads - 1;
    while (lo < hi) { const uint32_t mid = (lo + hi + 1) / 2; if (u0 >= p.sum0[mid]) lo = mid; else hi = mid - 1; }
    const uint32_t per_head = (p.sum0[lo + 1] - p.sum0[lo]) / p.n_kv, w = u0 - p.sum0[lo], kvh = w / per_head;
    const uint32_t hg = tid >> 6, r0 = (w % per_head) * kSumRows + (tid & 63) * 4;     // this thread's heads: hg, hg + 4, ...; its rows
    uint32_t item = p.lead[lo], most = 0;
    for (uint32_t i = item; i != 255; i = p.next[i]) most = max(most, p.rows[i]);
    float* sums = p.sums + ((uint64_t)p.seq[item] * p.n_kv + kvh) * p.max_seq + r0;
    float old[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) old[e] = hg == 0 && r0 + e < most ? sums[e] : 0.f;
    float4 add = make_float4(0.f, 0.f, 0.f, 0.f);
    for (; item != 255; item = p.next[item]) {
      const uint32_t ns = p.p_recs + p.n_own[item], rows = p.rows[item], pad = (rows + 63) & ~63u;
      const float* sc = p.scores + p.score0[item] + (uint64_t)kvh * p.G * pad + r0;
      constexpr int U = 4;
      float4 s[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r0 < rows && hg + 4 * u < p.G) s[u] = *reinterpret_cast<const float4*>(sc + (uint64_t)(hg + 4 * u) * pad);
      for (uint32_t h = warp; h < p.G; h += 8) {
        float M, l;
        shared_row_ml(reinterpret_cast<const float2*>(p.part_ml) + ((uint64_t)item * p.n_heads + kvh * p.G + h) * p.n_rec, ns, M, l);
        if (lane == 0) { s_m[h] = M; s_il[h] = __fdiv_rn(1.0f, l); }
      }
      __syncthreads();
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r0 < rows) {
        auto weigh = [&](const float4& v, uint32_t h) {
          const float m = s_m[h], il = s_il[h];
          t.x = fmaf(ex2_approx(fmaf(v.x, p.scale_log2, -m)), il, t.x); t.y = fmaf(ex2_approx(fmaf(v.y, p.scale_log2, -m)), il, t.y);
          t.z = fmaf(ex2_approx(fmaf(v.z, p.scale_log2, -m)), il, t.z); t.w = fmaf(ex2_approx(fmaf(v.w, p.scale_log2, -m)), il, t.w);
        };
#pragma unroll
        for (int u = 0; u < U; ++u) if (hg + 4 * u < p.G) weigh(s[u], hg + 4 * u);
        for (uint32_t h = hg + 4 * U; h < p.G; h += 4) weigh(*reinterpret_cast<const float4*>(sc + (uint64_t)h * pad), h);
      }
      s_acc[tid] = t;
      __syncthreads();
      if (hg == 0 && r0 < rows) {
#pragma unroll
        for (int i = 1; i < 4; ++i) { const float4 v = s_acc[tid + 64 * i]; t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w; }
        add.x += t.x;
        if (r0 + 1 < rows) add.y += t.y;
        if (r0 + 2 < rows) add.z += t.z;
        if (r0 + 3 < rows) add.w += t.w;
      }
    }
    if (hg == 0) {
      const float a[4] = {add.x, add.y, add.z, add.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) if (r0 + e < most) sums[e] = old[e] + a[e];
    }
  }
}

template <int HD, bool MIXED, bool FOLD>
static cudaError_t launch_shared_t(const SharedParams& p, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& k, const CUtensorMap& v, uint32_t n_kv,
                                   int dev, cudaStream_t st) {
  using S = ShSmem<HD>;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(pa_shared_kernel<HD, MIXED, FOLD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return e;
    attr_set[dev & 63].store(true, std::memory_order_release);
  }
  return launch_pdl(pa_shared_kernel<HD, MIXED, FOLD>, dim3(n_kv, p.units), dim3(S::THREADS), (size_t)S::TOTAL, st, pk, pv, k, v, p);
}
cudaError_t launch_shared(const SharedParams& p, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& k, const CUtensorMap& v, uint32_t hd, uint32_t n_kv,
                          int dev, cudaStream_t st) {
  const bool mixed = p.wide && p.p_splits, fold = p.fold > 1 || (mixed && p.p_tps > p.seg);      // (the other wide units leave one record)
  if (mixed && hd != 256) return cudaErrorInvalidValue;
  if (mixed) return fold ? launch_shared_t<256, true, true>(p, pk, pv, k, v, n_kv, dev, st) : launch_shared_t<256, true, false>(p, pk, pv, k, v, n_kv, dev, st);
  if (hd == 256) return fold ? launch_shared_t<256, false, true>(p, pk, pv, k, v, n_kv, dev, st) : launch_shared_t<256, false, false>(p, pk, pv, k, v, n_kv, dev, st);
  if (hd == 128) return fold ? launch_shared_t<128, false, true>(p, pk, pv, k, v, n_kv, dev, st) : launch_shared_t<128, false, false>(p, pk, pv, k, v, n_kv, dev, st);
  if (hd == 64) return fold ? launch_shared_t<64, false, true>(p, pk, pv, k, v, n_kv, dev, st) : launch_shared_t<64, false, false>(p, pk, pv, k, v, n_kv, dev, st);
  return cudaErrorInvalidValue;
}
cudaError_t launch_shared_finish(const SharedFinishParams& p, uint32_t hd, uint32_t sum_ctas, cudaStream_t st) {
  const dim3 grid(p.merge_ctas + sum_ctas);
  if (hd == 256) return sum_ctas ? launch_pdl(pa_shared_finish_kernel<256, true>, grid, dim3(256), 0, st, p) : launch_pdl(pa_shared_finish_kernel<256, false>, grid, dim3(256), 0, st, p);
  if (hd == 128) return sum_ctas ? launch_pdl(pa_shared_finish_kernel<128, true>, grid, dim3(256), 0, st, p) : launch_pdl(pa_shared_finish_kernel<128, false>, grid, dim3(256), 0, st, p);
  if (hd == 64) return sum_ctas ? launch_pdl(pa_shared_finish_kernel<64, true>, grid, dim3(256), 0, st, p) : launch_pdl(pa_shared_finish_kernel<64, false>, grid, dim3(256), 0, st, p);
  return cudaErrorInvalidValue;
}

}  // namespace pa
