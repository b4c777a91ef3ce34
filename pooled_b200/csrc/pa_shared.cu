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
  static_assert(!WIDE || HD == 256, "wide units");
  static constexpr int SB = WIDE || HD == 128 ? 2 : 3;      // tiles of scores in tensor memory; the weights take their scores' place
  static constexpr int TQC = WIDE ? 4 : HD == 256 ? 2 : 0;     // 64-dim chunks of Q in tensor memory, 32 columns each
  static constexpr int T_S = TQC * 32, T_O = T_S + SB * 64;
  static_assert(T_O + HD <= (HD == 256 ? 512 : 256), "tensor memory columns");
};
template <int HD>
constexpr int sh_tmem_cols() { return HD == 256 ? 512 : 256; }

enum { SH_K_FULL = 0, SH_K_EMPTY = 3, SH_V_FULL = 6, SH_V_EMPTY = 8, SH_S_FULL = 10, SH_P_FULL = 13, SH_PV_DONE = 16, SH_O_DONE = 19, SH_O_FREE, SH_Q_FULL, SH_Q_READ, SH_V_CLEAN, SH_BARS };
static_assert(SH_BARS <= 31, "barrier slots");

// a CTA's unit
struct ShUnit {
  const CUtensorMap* mk;
  const CUtensorMap* mv;
  uint32_t item0, slot, row0, n_rows, tile0, n_tiles;       // first item; record of a row; first row in the map; the unit's rows end here; its tiles
  uint32_t pairs, live_warps;                               // query rows; warps of a softmax group that hold them
  bool shared, ragged;                                      // shared rows; the last tile reaches past them
};

// warps 0 (K) and 3 (V), the same for both kinds of units; the tiles are read once, or by neighbouring CTAs at the same time, and
// enter L2 as its first to go
template <int HD>
__device__ __forceinline__ void shared_producer(const ShUnit& un, bool is_v, uint8_t* base, uint32_t bar0, volatile uint32_t* s_err) {
  using L = ShSmem<HD>;
  constexpr int CH = HD / 64;
  const uint32_t lane = threadIdx.x & 31, slots = is_v ? L::NV : L::NK, full = bar0 + 8 * (is_v ? SH_V_FULL : SH_K_FULL), empty = bar0 + 8 * (is_v ? SH_V_EMPTY : SH_K_EMPTY);
  uint8_t* ring = base + (is_v ? L::OFF_V : L::OFF_K);
  const CUtensorMap* map = is_v ? un.mv : un.mk;
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

// the other warps.  DIRECT: records of few rows may leave the lanes as they are; FOLD: all do, p.fold runs added up in each
template <int HD, bool WIDE, bool DIRECT, bool FOLD>
__device__ __forceinline__ void shared_roles(const SharedParams& p, const ShUnit& un, uint8_t* base, uint32_t bar0, volatile uint32_t* s_err, uint32_t tmem) {
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
      if (un.ragged && j == n_tiles - 1) mbar_wait(BAR(SH_V_CLEAN, 0), 0, s_err, WAIT_VFULL);
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
    if (!WIDE && p.scores && !un.shared && live) sc = p.scores + p.score0[un.item0] + ((uint64_t)g * G + lr) * ((un.n_rows + 63) & ~63u) + tile0 * 64 + mine;
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
      auto slot_of = [&](uint32_t pr) { const uint32_t it = row_item(pr); return ((uint64_t)(un.item0 + it) * p.n_heads + g * G + pr - it * G) * p.n_rec + un.slot + (FOLD ? seg / p.fold : seg); };
      if (!WIDE) l += __shfl_xor_sync(0xffffffffu, l, 1);
      float* sums = s_rl + (seg & 1) * 128 + row;          // two in turn: nothing else may come between two records
      if (wg) *sums = l;
      named_bar_sync(3 + qd, 64);
      if (!wg && live && !is_lo) {
        float2* ml = reinterpret_cast<float2*>(p.part_ml) + slot_of(lr);
        *ml = make_float2(m, FOLD && adds ? fmaf(ml->y, kept, l + *sums) : l + *sums);
      }
      constexpr uint32_t XW = WIDE ? 2 * L::X_BYTES : L::X_BYTES;
      static_assert(HD / 32 * XW <= (NK + NV) * L::KV_BYTES, "a place in the rings for every chunk");
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
        float* xs = reinterpret_cast<float*>(base + L::OFF_K + c * XW);
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
          if (kv0 + 64 > un.n_rows) {
#pragma unroll
            for (int i = 0; i < NS; ++i) if (kv0 + mine + i >= un.n_rows) s[i] = -INFINITY;
          }
          float mt = s[0];
#pragma unroll
          for (int i = 1; i < NS; ++i) mt = fmaxf(mt, s[i]);
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
          uint32_t hi[NS / 2], lo[NS / 2];
#pragma unroll
          for (int i = 0; i < NS / 2; ++i) {
            const float e0 = ex2_approx(fmaf(s[2 * i], p.scale_log2, -m_st)), e1 = ex2_approx(fmaf(s[2 * i + 1], p.scale_log2, -m_st));
            l_sum += e0 + e1;
            const __half2 h = __floats2half2_rn(e0, e1);
            const float2 f = __half22float2(h);
            hi[i] = *reinterpret_cast<const uint32_t*>(&h); lo[i] = pack_h2(e0 - f.x, e1 - f.y);
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
    }
  }
}

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
  // (m, l) of a row from its records, the same in every lane of the warp
  auto row_ml = [&](const float2* ml, uint32_t ns, float& M, float& l) {
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
  };
  pdl_wait();
  pdl_trigger();
  if (!SUMS || blockIdx.x < p.merge_ctas) {
    const uint32_t slices = HD / 4 / p.lanes, prow = blockIdx.x / slices, slice = blockIdx.x % slices, item = prow / p.n_heads, h = prow % p.n_heads;
    const uint32_t ns = p.p_recs + p.n_own[item], groups = 256 / p.lanes, grp = tid / p.lanes, ln = tid % p.lanes, dims = p.lanes * 4, d = slice * dims + tid;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + (uint64_t)prow * p.n_rec;
    const float* ob = p.part_o + (uint64_t)prow * p.n_rec * HD + slice * dims + ln * 4;
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
    row_ml(ml, ns, M, l);
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
        row_ml(reinterpret_cast<const float2*>(p.part_ml) + ((uint64_t)item * p.n_heads + kvh * p.G + h) * p.n_rec, ns, M, l);
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
