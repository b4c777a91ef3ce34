// Attention of trees of drafted tokens over a cache (pa_decode_tree).
//
//   o_c = sum_r e^(q_c.k_r / sqrt(hd) - M) v_r / sum_r e^(q_c.k_r / sqrt(hd) - M),   r < base, or r - base one of token c's ancestors or c itself
//
// A unit is a run of 64-row K / V tiles of one sequence and kv head, and a row tile: the group's heads of some of the tree's
// tokens.  Its CTA is the one of the shared-prefix decode (pa_shared.cuh: roles, precision, narrow and wide row tiles, records),
// and the tree's rows are simply the last of the sequence's, so a small tree costs one tile at most.  What the tree adds:
//   the mask    in tiles that hold rows of the tree a lane walks its token's parents (in shared memory, 35 cycles each, ahead of
//               the wait for the scores) and collects a bit for each of the tile's keys; scores of the other keys are -infinity by
//               selection, so whatever the K of a token that is no ancestor holds stays out
//   V           a weight of zero does not make up for an infinity or NaN: the V producer looks through the tree's rows of a tile
//               while the scores are being made, puts zeros in the place of such values and notes their rows; a token that attends
//               one of them has its values added to its record at the end, so that it ends as the formula does
// What bounds it: with few tokens HBM; from some 100 query rows a kv head on the issue of the tensor instructions, whose N is a tile's 64
// keys (with half of the L2 traffic taken away nothing changes): 64 tokens of 16 / 2 heads of 256 behind 32768 rows 52 us (0.40 of the
// measured rate of plain bf16 products), 16 x 60 of 16 / 8 heads of 128 behind up to 4003 rows 41 us, 6 x 26 of 24 / 4 heads of 256 with f32
// queries behind up to 9001 rows 58 us; 8 tokens behind 301 rows 7.5 us.  (At a sustained load the clock falls to 1.5 GHz: 61, 45 and 69 us.
// Tiles of 128 keys need one CTA an SM and the exponentials of a tile are then not hidden: 49, 45 and 55 us with 16 softmax warps, 59, 47 and
// 67 sustained, and 8.2 us for the 8 tokens.  Merged by the last CTA of each row tile instead of a second kernel: 11.4, 133, 85 and 56 us.)
#include "pa_shared.cuh"

namespace pa {

// grid (kv heads, units)
template <int HD, bool WIDE, bool FOLD>
__global__ void __launch_bounds__(384, ShSmem<HD>::CTAS)
pa_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TreeParams p) {
  using L = ShSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::OFF_BAR);
  volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(bars + 31);
  volatile uint32_t* s_err = s_tmem + 1;
  const uint32_t bar0 = smem_u32(bars);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t it = 0, hi = p.n_items - 1, u = blockIdx.y;
  while (it < hi) { const uint32_t mid = (it + hi + 1) / 2; if (u >= p.unit0[mid]) it = mid; else hi = mid - 1; }
  u -= p.unit0[it];
  const uint32_t rts = p.row_tiles[it], split = u / rts, rt = u - split * rts, c0 = rt * p.tile_cols[it];
  TreeUnit un;
  un.mk = &tm_k; un.mv = &tm_v;
  un.shared = un.ragged = false;
  un.item0 = p.col0[it] + c0;
  un.pairs = min((uint32_t)p.tile_cols[it], p.cols[it] - c0) * p.G;
  un.row0 = p.seq[it] * p.max_seq; un.n_rows = p.rows[it];
  un.tile0 = split * p.tps;
  un.n_tiles = min((un.n_rows + 63) / 64, un.tile0 + p.tps) - un.tile0;
  un.slot = un.tile0 / (FOLD ? p.seg * p.fold : p.seg);
  un.live_warps = ((WIDE ? 1 : 2) * un.pairs + 31) / 32;
  un.n_rec = p.n_rec[it]; un.rec0 = p.rec0[it] - (uint64_t)p.col0[it] * p.n_heads * un.n_rec;
  un.tree0 = p.base[it]; un.node0 = p.node0[it] + c0; un.parent0 = p.parent0[it];
  un.tree_tile = min(un.n_tiles, max(un.tree0 / 64, un.tile0) - un.tile0);

  if (warp == 1 && lane == 0) {
    *s_err = 0;
    auto init = [&](int which, int n, uint32_t count) { for (int i = 0; i < n; ++i) mbar_init(bar0 + 8u * (uint32_t)(which + i), count); };
    init(SH_K_FULL, 3, 1); init(SH_K_EMPTY, 3, 1); init(SH_V_FULL, 2, 1); init(SH_V_EMPTY, 2, 1);
    init(SH_S_FULL, 3, 1); init(SH_P_FULL, 3, 64 * un.live_warps); init(SH_PV_DONE, 3, 1);
    init(SH_O_DONE, 1, 1); init(SH_O_FREE, 1, 64 * un.live_warps); init(SH_Q_FULL, 1, 256); init(SH_Q_READ, 1, 256); init(SH_V_CLEAN, 2, 1);
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
  if (warp == 0 || warp == 3) shared_producer<HD, true>(un, warp == 3, base, bar0, s_err);
  else shared_roles<HD, WIDE, !WIDE, FOLD, true>(p, un, base, bar0, s_err, tmem);
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, sh_tmem_cols<HD>());
  }
  if (tid == 0 && *s_err) atomicMax(p.err, *s_err);
}

__device__ __forceinline__ uint32_t tree_item(const TreeFinishParams& p, uint32_t col) {
  uint32_t lo = 0, hi = p.n_items - 1;
  while (lo < hi) { const uint32_t mid = (lo + hi + 1) / 2; if (col >= p.col0[mid]) lo = mid; else hi = mid - 1; }
  return lo;
}

// Merge, gate, store.  Few rows: a CTA a row (or slice), as behind a shared prefix.  Many: a warp a piece of a row, eight a CTA, so that a
// row of two or three records does not take a CTA's start and two barriers.  (Pieces of 64 dims, half a warp on every other record: no faster
// with 1024 rows of 18 records, 3 to 6 us slower with thousands of rows.)
template <int HD, bool WARPS>
__global__ void __launch_bounds__(256, 4) pa_tree_finish_kernel(const __grid_constant__ TreeFinishParams p) {
  pdl_wait();
  pdl_trigger();
  if constexpr (!WARPS) {
    __shared__ float4 s_acc[256];
    const uint32_t slices = HD / 4 / p.lanes, prow = blockIdx.x / slices, col = prow / p.n_heads, it = tree_item(p, col);
    shared_merge_row<HD>(p, s_acc, p.rec0[it] + (uint64_t)(prow - p.col0[it] * p.n_heads) * p.n_rec[it], blockIdx.x % slices, col, prow % p.n_heads, p.n_rec[it]);
  } else {
    constexpr int PIECE = HD == 64 ? 64 : 128, PIECES = HD / PIECE, SIDES = 128 / PIECE, U = 8;       // dims; warps of a row; records of a load; loads at once
    const uint32_t w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, prow = w / PIECES, side = SIDES == 2 ? lane >> 4 : 0,
                   d = w % PIECES * PIECE + (SIDES == 2 ? lane & 15 : lane) * 4;
    if (prow >= p.n_rows) return;
    const uint32_t col = prow / p.n_heads, h = prow - col * p.n_heads, it = tree_item(p, col), ns = p.n_rec[it];
    const uint64_t rec = p.rec0[it] + (uint64_t)(prow - p.col0[it] * p.n_heads) * ns;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + rec;
    const float* ob = p.part_o + rec * HD + d;
    float4 x[U], acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto load = [&](uint32_t s0) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint32_t s = s0 + k * SIDES + side;
        x[k] = s < ns ? *reinterpret_cast<const float4*>(ob + (uint64_t)s * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    load(0);
    const uint64_t go = (uint64_t)col * p.gate_col_stride + (uint64_t)h * p.gate_head_stride + d, oo = (uint64_t)col * p.out_col_stride + (uint64_t)h * HD + d;
    float gv[4];
    if (p.gate) {
      if (p.vec && p.act_f16) {
        const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(p.gate) + go);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        gv[0] = a.x; gv[1] = a.y; gv[2] = b.x; gv[3] = b.y;
      } else if (p.vec) {
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.gate) + go);
        gv[0] = v.x; gv[1] = v.y; gv[2] = v.z; gv[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) gv[e] = ld_act(p.gate, go + e, p.act_f16);
      }
    }
    float M, l;
    shared_row_ml(ml, ns, M, l);
    for (uint32_t s0 = 0; s0 < ns; s0 += U * SIDES) {
      if (s0) load(s0);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint32_t s = s0 + k * SIDES + side;
        const float wt = s < ns ? ex2_approx(ml[s].x - M) : 0.f;
        acc.x = fmaf(x[k].x, wt, acc.x); acc.y = fmaf(x[k].y, wt, acc.y); acc.z = fmaf(x[k].z, wt, acc.z); acc.w = fmaf(x[k].w, wt, acc.w);
      }
    }
    float t[4] = {acc.x, acc.y, acc.z, acc.w};
    if constexpr (SIDES == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] += __shfl_down_sync(0xffffffffu, t[e], 16);
      if (side) return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = __fdiv_rn(t[e], l);
      if (p.gate) t[e] *= __fdiv_rn(1.0f, 1.0f + __expf(-gv[e]));
    }
    if (p.vec && p.act_f16) {
      const __half2 a = __floats2half2_rn(t[0], t[1]), b = __floats2half2_rn(t[2], t[3]);
      *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + oo) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else if (p.vec) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + oo) = make_float4(t[0], t[1], t[2], t[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (p.act_f16) reinterpret_cast<__half*>(p.out)[oo + e] = __float2half_rn(t[e]);
        else reinterpret_cast<float*>(p.out)[oo + e] = t[e];
      }
    }
  }
}

template <int HD, bool WIDE, bool FOLD>
static cudaError_t launch_tree_t(const TreeParams& p, const CUtensorMap& k, const CUtensorMap& v, uint32_t n_kv, int dev, cudaStream_t st) {
  using S = ShSmem<HD>;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(pa_tree_kernel<HD, WIDE, FOLD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return e;
    attr_set[dev & 63].store(true, std::memory_order_release);
  }
  return launch_pdl(pa_tree_kernel<HD, WIDE, FOLD>, dim3(n_kv, p.units), dim3(S::THREADS), (size_t)S::TOTAL, st, k, v, p);
}
template <int HD>
static cudaError_t launch_tree_h(const TreeParams& p, bool wide, const CUtensorMap& k, const CUtensorMap& v, uint32_t n_kv, int dev, cudaStream_t st) {
  const bool fold = p.fold > 1 || (wide && p.tps > p.seg);      // (wide units leave one record, or the sum of several runs)
  if (wide) return fold ? launch_tree_t<HD, true, true>(p, k, v, n_kv, dev, st) : launch_tree_t<HD, true, false>(p, k, v, n_kv, dev, st);
  return fold ? launch_tree_t<HD, false, true>(p, k, v, n_kv, dev, st) : launch_tree_t<HD, false, false>(p, k, v, n_kv, dev, st);
}
cudaError_t launch_tree(const TreeParams& p, bool wide, const CUtensorMap& k, const CUtensorMap& v, uint32_t hd, uint32_t n_kv, int dev, cudaStream_t st) {
  return hd == 256 ? launch_tree_h<256>(p, wide, k, v, n_kv, dev, st) : hd == 128 ? launch_tree_h<128>(p, wide, k, v, n_kv, dev, st)
       : hd == 64 ? launch_tree_h<64>(p, wide, k, v, n_kv, dev, st) : cudaErrorInvalidValue;
}
template <int HD>
static cudaError_t launch_finish_t(const TreeFinishParams& p, cudaStream_t st) {
  if (p.lanes) return launch_pdl(pa_tree_finish_kernel<HD, false>, dim3(p.n_rows * (HD / 4 / p.lanes)), dim3(256), 0, st, p);
  return launch_pdl(pa_tree_finish_kernel<HD, true>, dim3((p.n_rows * (HD == 256 ? 2 : 1) + 7) / 8), dim3(256), 0, st, p);
}
cudaError_t launch_tree_finish(const TreeFinishParams& p, uint32_t hd, cudaStream_t st) {
  return hd == 256 ? launch_finish_t<256>(p, st) : hd == 128 ? launch_finish_t<128>(p, st) : hd == 64 ? launch_finish_t<64>(p, st) : cudaErrorInvalidValue;
}

}  // namespace pa
