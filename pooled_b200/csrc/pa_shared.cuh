// The units of the shared-prefix, weighing and tree decodes: what the warps of a CTA that walks a run of K / V tiles do (the figures and the
// split stand in pa_shared.cu), and the merge of a row's records.
#pragma once
#include <algorithm>

#include "pa_tc.cuh"

namespace pa {

template <int HD>
struct ShSmem {
  // head_dim 128 and 64: two CTAs an SM (80 registers, 256 columns of tensor memory, 102 KB), so that one fetches, starts or stores while
  // the other multiplies
  static constexpr int CTAS = HD == 256 ? 1 : 2;
  static constexpr int NK = HD == 128 ? 2 : 3, NV = 2;
  static constexpr int KV_BYTES = HD * 128;          // [HD/64][64 rows][128 B]
  static constexpr int THREADS = 384;
  static constexpr int OFF_K = 0, OFF_V = NK * KV_BYTES, OFF_BAR = (NK + NV) * KV_BYTES;
  static constexpr int OFF_MAX = OFF_BAR + 256;      // [2][2][128] maxima of the rows, two tiles in turn, and [2][128] row sums
  static constexpr int OFF_Q = OFF_BAR + 4096;       // the chunks of Q that are not in tensor memory: two, of head_dim 64 one (narrow only)
  static constexpr int TOTAL = 1024 + OFF_Q + (HD == 64 ? 1 : 2) * 128 * 128;
  static_assert(CTAS * (TOTAL + 1024) <= 228 * 1024, "shared memory of an SM");
  static constexpr int XP = 36;                      // a chunk of a record on its way out through the rings: 64 or 128 rows of 32 floats, 36 apart
  static constexpr int X_BYTES = 64 * XP * 4;
};
template <int HD, bool WIDE>
struct ShLay {
  static constexpr int SB = WIDE || HD == 128 ? 2 : 3;      // tiles of scores in tensor memory; the weights take their scores' place
  static constexpr int TQC = HD != 256 ? 0 : WIDE ? 4 : 2;     // 64-dim chunks of Q in tensor memory, 32 columns each
  static constexpr int T_S = TQC * 32, T_O = T_S + SB * 64;
  static_assert(T_O + HD <= (HD == 256 ? 512 : 256), "tensor memory columns");
};
// rows of a tree of drafted tokens (a unit of pa_tree_kernel), behind the maxima and sums: every token's parent, i16, and the rows of up to five
// tiles whose V holds a value that is no finite number
constexpr int kTreeNodes = 256, kTreeTiles = kTreeNodes / 64 + 1;
constexpr int OFF_TREE = 256 + 3072, OFF_DIRTY = OFF_TREE + kTreeNodes * 2;       // from OFF_BAR on
static_assert(OFF_DIRTY + kTreeTiles * 8 + 4 <= 4096, "room behind the barriers");
template <int HD>
constexpr int sh_tmem_cols() { return HD == 256 ? 512 : 256; }

enum { SH_K_FULL = 0, SH_K_EMPTY = 3, SH_V_FULL = 6, SH_V_EMPTY = 8, SH_S_FULL = 10, SH_P_FULL = 13, SH_PV_DONE = 16, SH_O_DONE = 19, SH_O_FREE, SH_Q_FULL, SH_Q_READ, SH_V_CLEAN, SH_BARS = SH_V_CLEAN + 2 };
static_assert(SH_BARS <= 31, "barrier slots");

// a CTA's unit
struct ShUnit {
  const CUtensorMap* mk;
  const CUtensorMap* mv;
  uint32_t item0, slot, row0, n_rows, tile0, n_tiles;       // first item; record of a row; first row in the map; the unit's rows end here; its tiles
  uint32_t pairs, live_warps;                               // query rows; warps of a softmax group that hold them
  bool shared, ragged;                                      // shared rows; the last tile reaches past them
};
// ... of a tree: the rows from tree0 on are its tokens
struct TreeUnit : ShUnit {
  uint32_t tree0, node0, tree_tile, parent0;                // first row of the tree; token of the first query row; first tile (of the unit) that holds some; its parents
  uint32_t n_rec; uint64_t rec0;                            // records of a query row; where those of column 0, head 0 would be
};

// Warp 3 of a tree's unit: a weight of zero does not make up for an infinity or NaN in the V of a token that is no ancestor, so such values of the
// tree's rows become zeros here, ahead of the products, and their rows are noted: who attends one gets its values back when the record
// is written (tree_restore).  Rows behind the tree are cleared.
template <int HD>
__device__ __forceinline__ void tree_v_producer(const TreeUnit& un, uint8_t* ring, uint32_t full, uint32_t empty, uint32_t bar0, volatile uint32_t* s_err) {
  using L = ShSmem<HD>;
  constexpr int CH = HD / 64, PER = CH * 8, STEP = 8;       // 16-byte units of a row; rounds of the warp at once
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t policy = l2_policy_evict_first();
  uint32_t* dirty = reinterpret_cast<uint32_t*>(ring - L::OFF_V + L::OFF_BAR + OFF_DIRTY);
  auto clean = [&](uint32_t j) {
    const uint32_t st = j % L::NV, kv0 = (un.tile0 + j) * 64, from = un.tree0 > kv0 ? un.tree0 - kv0 : 0, to = min(64u, un.n_rows - kv0);
    mbar_wait(full + 8 * st, (j / L::NV) & 1, s_err, WAIT_VFULL);
    uint8_t* tile = ring + st * L::KV_BYTES;
    auto unit = [&](uint32_t i) { return reinterpret_cast<uint4*>(tile + (i % PER / 8) * (64 * 128) + (i / PER) * 128 + (i & 7) * 16); };
    auto odd = [](uint32_t w) { return ((w & 0x7fff7fffu) + 0x04000400u) & 0x80008000u; };      // the top bit of each half that is an infinity or NaN
    uint32_t bad0 = 0, bad1 = 0;
    for (uint32_t i0 = from * PER; i0 < to * PER; i0 += 32 * STEP) {
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        const uint32_t i = i0 + k * 32 + lane;
        if (i < to * PER) { const uint4 x = *unit(i); any |= odd(x.x) | odd(x.y) | odd(x.z) | odd(x.w); }
      }
      if (__any_sync(0xffffffffu, any != 0)) {
        for (uint32_t k = 0; k < STEP; ++k) {
          const uint32_t i = i0 + k * 32 + lane;
          if (i >= to * PER) continue;
          __half* h = reinterpret_cast<__half*>(unit(i));
          for (int e = 0; e < 8; ++e)
            if (!isfinite(__half2float(h[e]))) {
              h[e] = __float2half_rn(0.f);
              if (i / PER < 32) bad0 |= 1u << (i / PER); else bad1 |= 1u << (i / PER - 32);
            }
        }
      }
    }
    for (uint32_t i = to * PER + lane; i < 64 * PER; i += 32) *unit(i) = make_uint4(0, 0, 0, 0);
    bad0 = __reduce_or_sync(0xffffffffu, bad0); bad1 = __reduce_or_sync(0xffffffffu, bad1);
    if (lane == 0) { dirty[2 * (j - un.tree_tile)] = bad0; dirty[2 * (j - un.tree_tile) + 1] = bad1; }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar0 + 8 * (SH_V_CLEAN + st));      // (a barrier a slot: the next tile's may come before this one is waited for)
  };
  for (uint32_t j = 0; j < un.n_tiles; ++j) {
    if (lane == 0) {
      if (j == L::NV - 1) mbar_wait(bar0 + 8 * SH_Q_READ, 0, s_err, WAIT_QFULL);
      mbar_wait(empty + 8 * (j % L::NV), ((j / L::NV) & 1) ^ 1, s_err, WAIT_EMPTY);
      mbar_expect_tx(full + 8 * (j % L::NV), L::KV_BYTES);
      tma_load_3d_hint(smem_u32(ring + (j % L::NV) * L::KV_BYTES), un.mv, 0, (int)(un.row0 + (un.tile0 + j) * 64), (int)(blockIdx.x * CH), full + 8 * (j % L::NV), policy);
    }
    __syncwarp();
    if (j > un.tree_tile) clean(j - 1);
  }
  if (un.n_tiles > un.tree_tile) clean(un.n_tiles - 1);
}

// the keys of a tile that token `c` of a tree attends: bit i is row kv0 + i
static __device__ __noinline__ uint64_t tree_sees(const int16_t* parents, uint32_t c, uint32_t tree0, uint32_t kv0) {
  uint64_t m = kv0 < tree0 ? (tree0 - kv0 < 64 ? (1ull << (tree0 - kv0)) - 1 : ~0ull) : 0;
  for (int a = (int)c; a >= 0; a = parents[a]) {             // (a parent comes before its token)
    const int at = (int)(tree0 + a - kv0);
    if (at < 0) break;
    if (at < 64) m |= 1ull << at;
  }
  return m;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The weights of 16 keys as f16 pairs, high and low parts, and their sum, two values an instruction.  The high part is the weight with the bits
// that f16 lacks cut off (exact but for weights below 2^-14, 2^-21 of the row's largest), the low part what that leaves.
__device__ __forceinline__ float tree_weights(const float* s, float scale, float m, uint32_t (&hi)[8], uint32_t (&lo)[8]) {
  const float2 k = make_float2(scale, scale), ref = make_float2(-m, -m);
  float2 sum = make_float2(0.f, 0.f);
  auto bits = [](const float2& v) { return *reinterpret_cast<const unsigned long long*>(&v); };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned long long x;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(bits(make_float2(s[2 * i], s[2 * i + 1]))), "l"(bits(k)), "l"(bits(ref)));
    const float2 f = *reinterpret_cast<const float2*>(&x), e = make_float2(ex2_approx(f.x), ex2_approx(f.y));
    const float2 h = make_float2(__uint_as_float(__float_as_uint(e.x) & 0xffffe000u), __uint_as_float(__float_as_uint(e.y) & 0xffffe000u));
    unsigned long long t, l;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(t) : "l"(bits(sum)), "l"(bits(e)));
    sum = *reinterpret_cast<const float2*>(&t);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(l) : "l"(bits(h)), "l"(bits(make_float2(-1.f, -1.f))), "l"(bits(e)));
    const float2 rest = *reinterpret_cast<const float2*>(&l);
    hi[i] = pack_h2(h.x, h.y); lo[i] = pack_h2(rest.x, rest.y);
  }
  return sum.x + sum.y;
}

// Adds the V values that were no finite numbers to the last records of a unit's query rows, record `rec` of each: thread `tid` of `threads`.
template <int HD, typename P>
__device__ __noinline__ void tree_restore(const P& p, TreeUnit un, const uint32_t* dirty, const int16_t* parents, uint32_t rec, uint32_t tid, uint32_t threads) {
  for (uint32_t i = tid; i < un.pairs * (HD / 4); i += threads) {
    const uint32_t pr = i / (HD / 4), d = i % (HD / 4) * 4, it = pr / p.G;
    float4* at = reinterpret_cast<float4*>(p.part_o + (un.rec0 + ((uint64_t)(un.item0 + it) * p.n_heads + blockIdx.x * p.G + pr - it * p.G) * un.n_rec + rec) * HD + d);
    float4 t = *at;
    for (uint32_t j = un.tree_tile; j < un.n_tiles; ++j) {
      const uint32_t kv0 = (un.tile0 + j) * 64;
      uint64_t m = dirty[2 * (j - un.tree_tile)] | ((uint64_t)dirty[2 * (j - un.tree_tile) + 1] << 32);
      if (m) m &= tree_sees(parents, un.node0 + it, un.tree0, kv0);
      for (; m; m &= m - 1) {
        const __half* v = p.v + (uint64_t)(un.row0 + kv0 + __ffsll((long long)m) - 1) * p.kv_dim + blockIdx.x * HD + d;
        auto value = [&](int e) { const float x = __half2float(v[e]); return isfinite(x) ? 0.f : x; };
        t.x += value(0); t.y += value(1); t.z += value(2); t.w += value(3);
      }
    }
    *at = t;
  }
}

// warps 0 (K) and 3 (V), the same for both kinds of units; the tiles are read once, or by neighbouring CTAs at the same time, and
// enter L2 as its first to go
template <int HD, bool TREE = false, typename U>
__device__ __forceinline__ void shared_producer(const U& un, bool is_v, uint8_t* base, uint32_t bar0, volatile uint32_t* s_err) {
  using L = ShSmem<HD>;
  constexpr int CH = HD / 64;
  const uint32_t lane = threadIdx.x & 31, slots = is_v ? L::NV : L::NK, full = bar0 + 8 * (is_v ? SH_V_FULL : SH_K_FULL), empty = bar0 + 8 * (is_v ? SH_V_EMPTY : SH_K_EMPTY);
  uint8_t* ring = base + (is_v ? L::OFF_V : L::OFF_K);
  const CUtensorMap* map = is_v ? un.mv : un.mk;
  if constexpr (TREE) {
    if (is_v) { tree_v_producer<HD>(un, ring, full, empty, bar0, s_err); return; }
  }
  if (lane == 0) {
    const uint64_t policy = l2_policy_evict_first();
    for (uint32_t j = 0, st = 0, u = 0; j < un.n_tiles; ++j) {
      if (j == slots - 1) mbar_wait(bar0 + 8 * SH_Q_READ, 0, s_err, WAIT_QFULL);      // the last slot stages query rows until then
      mbar_wait(empty + 8 * st, (u & 1) ^ 1, s_err, WAIT_EMPTY);
      mbar_expect_tx(full + 8 * st, L::KV_BYTES);
      tma_load_3d_hint(smem_u32(ring + st * L::KV_BYTES), map, 0, (int)(un.row0 + (un.tile0 + j) * 64), (int)(blockIdx.x * CH), full + 8 * st, policy);
      if (++st == slots) { st = 0; ++u; }
    }
  }
  __syncwarp();
  if (is_v && un.ragged) {
    const uint32_t j = un.n_tiles - 1, st = j % L::NV, from = un.n_rows - (un.tile0 + j) * 64;
    mbar_wait(full + 8 * st, (j / L::NV) & 1, s_err, WAIT_VFULL);
    for (uint32_t i = lane; i < (64 - from) * 8 * CH; i += 32) {
      const uint32_t c = i / ((64 - from) * 8), w = i % ((64 - from) * 8);
      *reinterpret_cast<uint4*>(ring + st * L::KV_BYTES + c * (64 * 128) + from * 128 + w * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar0 + 8 * SH_V_CLEAN);
  }
}

// the other warps.  DIRECT: records of few rows may leave the lanes as they are; FOLD: all do, p.fold runs added up in each; TREE: a query row is
// that of a token, and of the rows from un.tree0 on it attends its ancestors and itself
template <int HD, bool WIDE, bool DIRECT, bool FOLD, bool TREE = false, typename P, typename U>
__device__ __forceinline__ void shared_roles(const P& p, const U& un, uint8_t* base, uint32_t bar0, volatile uint32_t* s_err, uint32_t tmem) {
  using L = ShSmem<HD>;
  using T = ShLay<HD, WIDE>;
  constexpr int CH = HD / 64, NK = L::NK, NV = L::NV, SB = T::SB, GRP = 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t g = blockIdx.x, n_tiles = un.n_tiles, tile0 = un.tile0;
  auto BAR = [&](int which, int idx) { return bar0 + 8u * (uint32_t)(which + idx); };
  uint8_t* q_s = base + L::OFF_Q;
  const uint32_t t_q = tmem, t_s0 = tmem + T::T_S, t_o = tmem + T::T_O;

  if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer, scores ----
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc_qk = umma_idesc(128, 64, 0);
    const uint64_t k_desc = smem_desc(smem_u32(base + L::OFF_K), 16, 1024);
    const uint64_t q_desc = smem_desc(smem_u32(q_s), 16, 1024);
    mbar_wait(BAR(SH_Q_FULL, 0), 0, s_err, WAIT_QFULL);
    tc_fence_after();
    for (uint32_t j = 0; j < n_tiles; ++j) {
      const uint32_t sb = j % SB, st = j % NK;
      if (j >= (uint32_t)SB) mbar_wait(BAR(SH_PV_DONE, sb), ((j - SB) / SB) & 1, s_err, WAIT_MMA);
      mbar_wait(BAR(SH_K_FULL, st), (j / NK) & 1, s_err, WAIT_KFULL);
      tc_fence_after();
      const uint64_t kd = k_desc + (uint64_t)(st * (L::KV_BYTES >> 4));
      const uint32_t ts = t_s0 + sb * 64;
      auto k_at = [&](int ks) { return kd + (uint64_t)(((ks >> 2) * (64 * 128) + (ks & 3) * 32) >> 4); };
      auto q_at = [&](int ks) { return q_desc + (uint64_t)(((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4); };
      constexpr int TS = T::TQC * 4;           // the dims whose Q chunks sit in tensor memory
#pragma unroll
      for (int ks = 0; ks < TS; ++ks) umma_f16_ts(leader, ts, t_q + ks * 8, k_at(ks), idesc_qk, ks > 0);
#pragma unroll
      for (int ks = TS; ks < HD / 16; ++ks) umma_f16_ss(leader, ts, q_at(ks - TS), k_at(ks), idesc_qk, ks > 0 ? 1u : 0u);
      umma_commit_elected(leader, BAR(SH_K_EMPTY, st));
      umma_commit_elected(leader, BAR(SH_S_FULL, sb));
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ MMA issuer, P V ----
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc_pv = umma_idesc(128, HD, 1);
    const uint64_t v_desc = smem_desc(smem_u32(base + L::OFF_V), 64 * 128, 1024);
    for (uint32_t j = 0, seg = 0, in_seg = 0; j < n_tiles; ++j) {
      const uint32_t sb = j % SB, st = j % NV;
      mbar_wait(BAR(SH_P_FULL, sb), (j / SB) & 1, s_err, WAIT_QFULL);
      mbar_wait(BAR(SH_V_FULL, st), (j / NV) & 1, s_err, WAIT_VFULL);
      if constexpr (TREE) {
        if (j >= un.tree_tile) mbar_wait(BAR(SH_V_CLEAN, st), ((j - un.tree_tile) / NV) & 1, s_err, WAIT_VFULL);
      } else {
        if (un.ragged && j == n_tiles - 1) mbar_wait(BAR(SH_V_CLEAN, 0), 0, s_err, WAIT_VFULL);
      }
      if (in_seg == 0 && j > 0) mbar_wait(BAR(SH_O_FREE, 0), (seg - 1) & 1, s_err, WAIT_MMA);      // the record before is out
      tc_fence_after();
      const uint64_t vd = v_desc + (uint64_t)(st * (L::KV_BYTES >> 4));
      const uint32_t tp = t_s0 + sb * 64;      // P(j): packed f16 pairs over S(j): 32 columns, wide: 32 of high and 32 of low parts
#pragma unroll
      for (int ks = 0; ks < (WIDE ? 8 : 4); ++ks)
        umma_f16_ts(leader, t_o, tp + ks * 8, vd + (uint64_t)(((ks & 3) * 2048) >> 4), idesc_pv, (in_seg > 0 || ks > 0) ? 1u : 0u);
      umma_commit_elected(leader, BAR(SH_V_EMPTY, st));
      umma_commit_elected(leader, BAR(SH_PV_DONE, sb));
      if (++in_seg == p.seg || j == n_tiles - 1) {
        umma_commit_elected(leader, BAR(SH_O_DONE, 0));
        in_seg = 0; ++seg;
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue ----
    const uint32_t wg = (warp - 4) >> 2, qd = (warp - 4) & 3, row = qd * 32 + lane;
    const uint32_t lane_addr = (qd * 32) << 16;
    const bool is_lo = !WIDE && (row & 1u) != 0, in_use = qd < un.live_warps;
    const uint32_t lr = WIDE ? row : row >> 1;         // query row: (item, head of the group)
    const bool live = lr < un.pairs;
    const uint32_t st_tid = tid - 128, G = p.G, by_g = (65536 + G - 1) / G;
    auto row_item = [&](uint32_t pr) { return (pr * by_g) >> 16; };       // pr / G, pr < 128
    int16_t* parents = reinterpret_cast<int16_t*>(base + L::OFF_BAR + OFF_TREE);
    if constexpr (TREE) {
      // a parent that is no earlier token of the tree: none (a chain where there are no parents: every token's is the one before it)
      if (un.tree_tile < n_tiles && st_tid < un.n_rows - un.tree0) {
        const int a = p.parents ? p.parents[un.parent0 + st_tid] : (int)st_tid - 1;
        parents[st_tid] = (int16_t)(a >= 0 && a < (int)st_tid ? a : -1);
      }
    }
    // The query rows come by cp.async into the last K and V slots, which the producers leave alone until Q_READ, half of them each, a
    // row's 16-byte chunks XOR-swizzled against the per-row reads.
    {
      const bool f16 = WIDE || p.q_f16;
      const uint32_t es = f16 ? 2u : 4u, cap = f16 ? 64u : 32u, q_ch = f16 ? HD / 8 : HD / 4;
      auto stage_row = [&](uint32_t r) { return base + (r < cap ? L::OFF_K + (NK - 1) * L::KV_BYTES : L::OFF_V + (NV - 1) * L::KV_BYTES) + (size_t)(r & (cap - 1)) * (HD * es); };
      for (uint32_t idx = st_tid; idx < un.pairs * q_ch; idx += 128 * GRP) {
        const uint32_t pr = idx / q_ch, c = idx % q_ch, it = row_item(pr);
        const uint8_t* src = reinterpret_cast<const uint8_t*>(p.q) +
                             ((uint64_t)(un.item0 + it) * p.q_col_stride + (uint64_t)(g * G + pr - it * G) * p.q_head_stride) * es + (uint64_t)c * 16;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(stage_row(pr) + ((c ^ (pr & 7u)) << 4))), "l"(src) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      named_bar_sync(1, 128 * GRP);
      const uint8_t* my_stage = stage_row(lr);
      auto stage_ld = [&](uint32_t c) { return live ? *reinterpret_cast<const uint4*>(my_stage + ((c ^ (lr & 7u)) << 4)) : make_uint4(0, 0, 0, 0); };
      // this thread's Q row as f16 pairs, 64 dims at a time (the groups share the chunks out)
#pragma unroll 1
      for (int c = 0; c < CH; ++c) {
        if (!in_use || (CH >= 2 ? (uint32_t)(c >= CH / 2) != wg : wg != 0)) continue;     // (rows without a query: whatever is there)
        uint32_t w[32];
        if (f16) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 x = is_lo ? make_uint4(0, 0, 0, 0) : stage_ld(c * 8 + i);         // f16 queries have no low part
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint4 r4 = stage_ld(c * 16 + i);
            float4 x = *reinterpret_cast<const float4*>(&r4);
            if (is_lo) {                                                                  // what the high part leaves over
              x.x -= __half2float(__float2half_rn(x.x)); x.y -= __half2float(__float2half_rn(x.y));
              x.z -= __half2float(__float2half_rn(x.z)); x.w -= __half2float(__float2half_rn(x.w));
            }
            w[2 * i] = pack_h2(x.x, x.y); w[2 * i + 1] = pack_h2(x.z, x.w);
          }
        }
        if (c < T::TQC) {
          tmem_st32u(t_q + c * 32 + lane_addr, w);
        } else {
          uint8_t* dst = q_s + (c - T::TQC) * (128 * 128) + row * 128;
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(dst + ((i ^ (row & 7)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      }
    }
    fence_proxy_async();
    mbar_arrive(BAR(SH_Q_READ, 0));
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(BAR(SH_Q_FULL, 0));

    // Both groups work on the same tile: of this lane's row the 32 keys of its group (narrow: shared with the row's other lane, 16 each).
    constexpr int NS = WIDE ? 32 : 16;
    const uint32_t mine = wg * 32 + (is_lo ? 16 : 0);     // this lane's first key of a tile
    float m_st = -1.0e30f, l_sum = 0.f;
    float* sc = nullptr;                                  // where the scores of this lane's keys go
    if constexpr (!TREE) if (!WIDE && p.scores && !un.shared && live) sc = p.scores + p.score0[un.item0] + ((uint64_t)g * G + lr) * ((un.n_rows + 63) & ~63u) + tile0 * 64 + mine;
    // the maximum of a row over both groups, whose warps of the same rows meet at a barrier of their own; two buffers in turn
    float* s_max = reinterpret_cast<float*>(base + L::OFF_MAX);
    auto row_max = [&](float m, uint32_t j) {
      tc_fence_before();                                  // this warp's scores have been read: the other's weights may take their place
      float* at = s_max + (j & 1) * 256 + row;
      at[wg * 128] = m;
      named_bar_sync(3 + qd, 64);
      tc_fence_after();
      return fmaxf(m, at[(wg ^ 1) * 128]);
    };
    // The record of the tiles since the last one.  Of up to 16 query rows, or while the rings are in use, the lanes store what they have, 64
    // bytes of a chunk of 32 dims (or add it to what they stored there before); else a unit's only or last record goes through the rings, idle by then, so that whole lines leave
    // (a lane has a row: its own stores are 16 bytes each in 32 records 1 KB apart).
    float* s_rl = s_max + 512;
    float m_rec = 0.f;                                    // the reference of what the lane has stored so far in a record of several runs
    auto record = [&](uint32_t seg, float m, float l, bool last) {
      const bool adds = FOLD && seg % p.fold != 0;
      const float kept = adds ? ex2_approx(m_rec - m) : 0.f;
      const uint32_t threads = 32 * un.live_warps, gt = (tid - 128) & 127;
      auto slot_of = [&](uint32_t pr) {
        const uint32_t it = row_item(pr);
        const uint64_t row = (uint64_t)(un.item0 + it) * p.n_heads + g * G + pr - it * G;
        if constexpr (TREE) return un.rec0 + row * un.n_rec + un.slot + (FOLD ? seg / p.fold : seg);
        else return row * p.n_rec + un.slot + (FOLD ? seg / p.fold : seg);
      };
      if (!WIDE) l += __shfl_xor_sync(0xffffffffu, l, 1);
      float* sums = s_rl + (seg & 1) * 128 + row;          // two in turn: nothing else may come between two records
      if (wg) *sums = l;
      named_bar_sync(3 + qd, 64);
      if (!wg && live && !is_lo) {
        float2* ml = reinterpret_cast<float2*>(p.part_ml) + slot_of(lr);
        *ml = make_float2(m, FOLD && adds ? fmaf(ml->y, kept, l + *sums) : l + *sums);
      }
      constexpr uint32_t XW = WIDE ? 2 * L::X_BYTES : L::X_BYTES;
      constexpr int PLACES = HD / 32 * XW <= (NK + NV) * L::KV_BYTES ? HD / 32 : GRP;      // a place in the rings for every chunk, or one for each group
      static_assert(PLACES * XW <= (NK + NV) * L::KV_BYTES, "places in the rings");
      mbar_wait(BAR(SH_O_DONE, 0), seg & 1, s_err, WAIT_MMA);
      tc_fence_after();
      // high and low rows of a chunk added, each lane with half of it
      auto add_rows = [&](const float* o, float (&t)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float give = is_lo ? o[i] : o[16 + i], keep = is_lo ? o[16 + i] : o[i];
          t[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
        }
      };
      if (FOLD || (DIRECT && (un.live_warps == 1 || !last))) {
        constexpr int N = HD == 256 ? 2 : 1, E = WIDE ? 32 : 16;              // chunks at a time; values of a chunk that a lane stores
        float* to = p.part_o + slot_of(live ? lr : 0) * HD + (is_lo ? 16 : 0);
#pragma unroll 1
        for (int c = wg; c < HD / 32; c += N * GRP) {
          float o[32 * N];
#pragma unroll
          for (int k = 0; k < N; ++k) tmem_ld32_async(t_o + (c + k * GRP) * 32 + lane_addr, o + 32 * k);
          tmem_wait_ld(o);
#pragma unroll
          for (int k = 0; k < N; ++k) {
            float t[E];
            if constexpr (WIDE) {
#pragma unroll
              for (int i = 0; i < E; ++i) t[i] = o[32 * k + i];
            } else {
              add_rows(o + 32 * k, t);
            }
            float4* at = reinterpret_cast<float4*>(to + (c + k * GRP) * 32);
            if (FOLD && live && adds) {
#pragma unroll
              for (int i = 0; i < E; i += 4) {
                const float4 x = at[i / 4];
                t[i] = fmaf(x.x, kept, t[i]); t[i + 1] = fmaf(x.y, kept, t[i + 1]); t[i + 2] = fmaf(x.z, kept, t[i + 2]); t[i + 3] = fmaf(x.w, kept, t[i + 3]);
              }
            }
            if (live) {
#pragma unroll
              for (int i = 0; i < E; i += 4) at[i / 4] = make_float4(t[i], t[i + 1], t[i + 2], t[i + 3]);
            }
          }
        }
        m_rec = m;
        tc_fence_before();
        mbar_arrive(BAR(SH_O_FREE, 0));
        return;
      }
#pragma unroll 1
      for (int c = wg; c < HD / 32; c += GRP) {           // the groups share the chunks out
        float o[32];
        tmem_ld32(t_o + c * 32 + lane_addr, o);
        float* xs = reinterpret_cast<float*>(base + L::OFF_K + c % PLACES * XW);
        if (PLACES < HD / 32 && c >= GRP) named_bar_sync(7 + wg, threads);      // the chunk before has left its place
        if constexpr (WIDE) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(xs + row * L::XP + 4 * i) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else {
          float t[16];
          add_rows(o, t);
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(xs + lr * L::XP + (is_lo ? 16 : 0) + 4 * i) = make_float4(t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]);
        }
        named_bar_sync(7 + wg, threads);
        for (uint32_t i = gt; i < un.pairs * 8; i += threads)
          reinterpret_cast<float4*>(p.part_o + slot_of(i >> 3) * HD + c * 32)[i & 7] = *reinterpret_cast<const float4*>(xs + (i >> 3) * L::XP + (i & 7) * 4);
      }
      tc_fence_before();
    };
    if (in_use) {
      float m_old = -3.0e30f, l_old = 0.f;                // of the record to be written next (m below -2e30: none)
      for (uint32_t j = 0, seg = 0, in_seg = 0;; ++j) {
        if (j < n_tiles) {
          const uint32_t b = j % SB, u = j / SB, kv0 = (tile0 + j) * 64;
          uint32_t sees = 0xffffffffu;                     // which of its keys this lane's row attends
          if constexpr (TREE) {
            if (j >= un.tree_tile) sees = live ? (uint32_t)(tree_sees(parents, un.node0 + row_item(lr), un.tree0, kv0) >> mine) : 0;
          }
          mbar_wait(BAR(SH_S_FULL, b), u & 1, s_err, WAIT_MMA);
          tc_fence_after();
          float s[NS];
          if constexpr (WIDE) {
            tmem_ld32(t_s0 + b * 64 + wg * 32 + lane_addr, s);
          } else {
            // a lane sends the half of its row (high or low parts) that the other lane has the keys of, and adds what comes back to its own
            float t[32];
            tmem_ld32(t_s0 + b * 64 + wg * 32 + lane_addr, t);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float give = is_lo ? t[i] : t[16 + i], keep = is_lo ? t[16 + i] : t[i];
              s[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
            }
          }
          if (!WIDE && sc) {
            float4* d = reinterpret_cast<float4*>(sc + j * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
          }
          if constexpr (TREE) {
            if (j >= un.tree_tile) {
#pragma unroll
              for (int i = 0; i < NS; ++i) if (!((sees >> i) & 1u)) s[i] = -INFINITY;
            }
          } else if (kv0 + 64 > un.n_rows) {
#pragma unroll
            for (int i = 0; i < NS; ++i) if (kv0 + mine + i >= un.n_rows) s[i] = -INFINITY;
          }
          float mt = s[0];
          if constexpr (TREE) {
            mt = fmaxf(mt, s[1]);
#pragma unroll
            for (int i = 2; i < NS; i += 2) mt = max3(mt, s[i], s[i + 1]);
          } else {
#pragma unroll
            for (int i = 1; i < NS; ++i) mt = fmaxf(mt, s[i]);
          }
          if (!WIDE) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
          mt = row_max(mt, j) * p.scale_log2;
          float alpha = 1.f;
          bool grow = false;
          if (mt > m_st + 15.f) { alpha = ex2_approx(m_st - (mt - 7.f)); m_st = mt - 7.f; l_sum *= alpha; grow = true; }
          if (in_seg > 0 && __any_sync(0xffffffffu, grow)) {
            const uint32_t jb = (j - 1) % SB, ju = (j - 1) / SB;
            mbar_wait(BAR(SH_PV_DONE, jb), ju & 1, s_err, WAIT_MMA);
            tc_fence_after();
#pragma unroll 1
            for (int c = wg; c < HD / 32; c += GRP) {       // the groups share the columns out
              float o[32];
              tmem_ld32(t_o + c * 32 + lane_addr, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= alpha;
              tmem_st32(t_o + c * 32 + lane_addr, o);
            }
          }
          // weights as f16 pairs, high and low parts
          if constexpr (TREE && WIDE) {                    // (16 keys at a time: two CTAs an SM have 80 registers a thread)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t hi[8], lo[8];
              l_sum += tree_weights(s + 16 * h, p.scale_log2, m_st, hi, lo);
              tmem_st8u(t_s0 + b * 64 + 16 * wg + 8 * h + lane_addr, hi);
              tmem_st8u(t_s0 + b * 64 + 32 + 16 * wg + 8 * h + lane_addr, lo);
            }
          } else {
            uint32_t hi[NS / 2], lo[NS / 2];
            if constexpr (TREE) {
              l_sum += tree_weights(s, p.scale_log2, m_st, hi, lo);
            } else {
#pragma unroll
              for (int i = 0; i < NS / 2; ++i) {
                const float e0 = ex2_approx(fmaf(s[2 * i], p.scale_log2, -m_st)), e1 = ex2_approx(fmaf(s[2 * i + 1], p.scale_log2, -m_st));
                l_sum += e0 + e1;
                const __half2 h = __floats2half2_rn(e0, e1);
                const float2 f = __half22float2(h);
                hi[i] = *reinterpret_cast<const uint32_t*>(&h); lo[i] = pack_h2(e0 - f.x, e1 - f.y);
              }
            }
            if constexpr (WIDE) {
              tmem_st16u(t_s0 + b * 64 + 16 * wg + lane_addr, hi);
              tmem_st16u(t_s0 + b * 64 + 32 + 16 * wg + lane_addr, lo);
            } else {
              // the even lane's row takes the high parts of the group's 32 keys, the odd one's the low parts
              uint32_t pw[16];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, is_lo ? hi[i] : lo[i], 1);
                pw[i] = is_lo ? got : hi[i];
                pw[8 + i] = is_lo ? lo[i] : got;
              }
              tmem_st16u(t_s0 + b * 64 + 16 * wg + lane_addr, pw);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(BAR(SH_P_FULL, b));
        }
        // a record is written behind the weights of the tile after its last, while the products of its last retire
        const bool last = j == n_tiles;
        if (last) { m_old = m_st; l_old = l_sum; }
        if (m_old > -2.0e30f) { record(seg++, m_old, l_old, last); m_old = -3.0e30f; }
        if (last) break;
        if (++in_seg == p.seg && j != n_tiles - 1) { m_old = m_st; l_old = l_sum; l_sum = 0.f; in_seg = 0; }
      }
      if constexpr (TREE) {
        const uint32_t* dirty = reinterpret_cast<const uint32_t*>(base + L::OFF_BAR + OFF_DIRTY);
        uint32_t any = 0;
        for (uint32_t i = 2 * un.tree_tile; i < 2 * n_tiles; ++i) any |= dirty[i - 2 * un.tree_tile];
        if (any) {
          const uint32_t last = (n_tiles - 1) / p.seg, threads = 64 * un.live_warps;
          named_bar_sync(1, threads);                       // the records are stored
          tree_restore<HD>(p, un, dirty, parents, un.slot + (FOLD ? last / p.fold : last), wg * 32 * un.live_warps + qd * 32 + lane, threads);
        }
      }
    }
  }
}

// (m, l) of a row from its records, the same in every lane of the warp
__device__ __forceinline__ void shared_row_ml(const float2* ml, uint32_t ns, float& M, float& l) {
  const uint32_t lane = threadIdx.x & 31;
  float2 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = lane + 32 * k < ns ? ml[lane + 32 * k] : make_float2(-3.0e38f, 0.f);
  M = fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x));
  for (uint32_t s = lane + 128; s < ns; s += 32) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  l = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) l = fmaf(v[k].y, ex2_approx(v[k].x - M), l);
  for (uint32_t s = lane + 128; s < ns; s += 32) { const float2 w = ml[s]; l = fmaf(w.y, ex2_approx(w.x - M), l); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
}
// one row (column, head) of `ns` records from `rec` on, or one slice of it, merged, gated and stored by a CTA of 256 threads
template <int HD, typename P>
__device__ __forceinline__ void shared_merge_row(const P& p, float4* s_acc, uint64_t rec, uint32_t slice, uint32_t item, uint32_t h, uint32_t ns) {
  const uint32_t tid = threadIdx.x, groups = 256 / p.lanes, grp = tid / p.lanes, ln = tid % p.lanes, dims = p.lanes * 4, d = slice * dims + tid;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + rec;
  const float* ob = p.part_o + rec * HD + slice * dims + ln * 4;
  constexpr int U = 4;      // (eight: two CTAs an SM, a second wave for 512 rows)
  float4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t s = grp + u * groups;
    x[u] = s < ns ? *reinterpret_cast<const float4*>(ob + (uint64_t)s * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float gv = 0.f;
  const bool gated = p.gate && tid < dims;
  if (gated) gv = ld_act(p.gate, (uint64_t)item * p.gate_col_stride + (uint64_t)h * p.gate_head_stride + d, p.act_f16);
  float M, l;
  shared_row_ml(ml, ns, M, l);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& r, uint32_t s) {
    const float w = s < ns ? ex2_approx(ml[s].x - M) : 0.f;
    acc.x = fmaf(r.x, w, acc.x); acc.y = fmaf(r.y, w, acc.y); acc.z = fmaf(r.z, w, acc.z); acc.w = fmaf(r.w, w, acc.w);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) add(x[u], grp + u * groups);
  for (uint32_t s0 = grp + U * groups; s0 < ns; s0 += U * groups) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t s = s0 + u * groups;
      x[u] = s < ns ? *reinterpret_cast<const float4*>(ob + (uint64_t)s * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) add(x[u], s0 + u * groups);
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < dims) {
    const float* sa = reinterpret_cast<const float*>(s_acc);
    float t = sa[tid];
    for (uint32_t i = 1; i < groups; ++i) t += sa[i * dims + tid];
    t = __fdiv_rn(t, l);
    if (gated) t *= __fdiv_rn(1.0f, 1.0f + __expf(-gv));
    const uint64_t oo = (uint64_t)item * p.out_col_stride + (uint64_t)h * HD + d;
    if (p.act_f16) reinterpret_cast<__half*>(p.out)[oo] = __float2half_rn(t);
    else reinterpret_cast<float*>(p.out)[oo] = t;
  }
}

}  // namespace pa
