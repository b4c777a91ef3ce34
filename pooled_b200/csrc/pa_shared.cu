// Attention of a batch of single tokens that share their first rows (pa_decode_shared), and of a batch whose weights are summed
// per cached row (pa_decode_weights): one kernel over both kinds of rows, and one that merges.
//
//   o = sum_r e^(q.k_r / sqrt(hd) - M) v_r / sum_r e^(q.k_r / sqrt(hd) - M)   over the shared rows and the item's own
//
// A unit is a run of 64-row K / V tiles of one kv head and up to 64 query rows that attend them: for the shared rows the
// heads of several items (so that each shared byte is read once per 64 query rows, from HBM once in all), for own rows the
// heads of one.  A CTA per unit walks its tiles on the 5th-generation tensor cores and leaves an unnormalised (o, m, l)
// record per query row; the second kernel merges a row's records, gates and stores.  All units have the same number of
// tiles, whatever they are units of (plan_shared), so that a batch of long shared rows and short own ones fills the
// machine like one long conversation.
//
//   warps 0, 3  TMA producers: K tiles and V tiles (64 x head_dim f16, 128-byte swizzle), a ring of three and of two slots;
//               warp 3 then clears the rows of the last V tile that lie behind the unit's last: a weight of zero does not
//               make up for an infinity or NaN that the cache holds there
//   warp 1      issues the scores: S = Q K^T into one of three tiles of tensor memory (128 x 64 f32)
//   warp 2      tensor memory; issues O += P V into the accumulator (128 x head_dim f32)
//   warps 4-11  two softmax groups on alternate tiles.  Even rows of the 128 carry the f16 high parts of q and of the
//               weights, odd rows the low parts of the same query row: some 22 bits of both, added by shuffles.  The two lanes
//               share the row's keys out (each with all 64, a tile took 2 us of a group instead of 1.2).  A row's reference lies 2^7 below its maximum, moves only when a tile passes it by 2^15, and travels
//               with the tiles: weights of up to 2^15 keep the low parts of small ones above f16's last place (with a
//               reference at the maximum, a long row's error was 2.2e-6 of the result, 3e-7 now).
//               Warps whose rows hold no query take no part.
// What bounds it: one query tile per kv head, HBM; several, the tensor cores (1394 cycles for both products of 64 keys at
// head_dim 256).
#include <algorithm>

#include "pa_tc.cuh"

namespace pa {

template <int HD>
struct ShSmem {
  static constexpr int SBUF = 3, NK = 3, NV = 2;
  static constexpr int KV_BYTES = HD * 128;          // [HD/64][64 rows][128 B]
  static constexpr int TQC = HD / 128;               // 64-dim chunks of Q in tensor memory, the others in shared memory
  static constexpr int QS_BYTES = (HD / 64 - TQC) * 128 * 128;
  static constexpr int THREADS = 384;
  static constexpr int OFF_K = 0, OFF_V = NK * KV_BYTES, OFF_Q = (NK + NV) * KV_BYTES, OFF_BAR = OFF_Q + QS_BYTES;
  static constexpr int OFF_ROW = OFF_BAR + 256;      // [128] reference maximum of each row
  static constexpr int TOTAL = 1024 + OFF_ROW + 128 * 4;
  static_assert(TOTAL <= 227 * 1024, "shared memory of one CTA");
  // the records leave through the K ring: row sums of the groups, then 64 rows of HD + 4 floats and their slots
  static_assert(2048 + 64 * (HD + 4) * 4 + 64 * 8 <= (NK + NV) * KV_BYTES, "staging of the records");
  static constexpr int T_Q = 0, T_S = TQC * 32, T_O = TQC * 32 + SBUF * 64;
  static constexpr int TMEM_COLS = T_O + HD <= 256 ? 256 : 512;
  static_assert(T_O + HD <= 512, "tensor memory columns");
};

template <int HD>
__global__ void __launch_bounds__(384, 1)
pa_shared_kernel(const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ SharedParams p) {
  using L = ShSmem<HD>;
  constexpr int CH = HD / 64, NK = L::NK, NV = L::NV, SB = L::SBUF, GRP = 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::OFF_BAR);
  volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(bars + 31);
  volatile uint32_t* s_err = s_tmem + 1;
  float* s_rm = reinterpret_cast<float*>(base + L::OFF_ROW);
  float* s_rl = reinterpret_cast<float*>(base + L::OFF_K);       // [2][128] the groups' row sums and [2][128] what they are expressed in,
  float* s_rr = s_rl + 256;                                      // in the first K slot once the last tile's scores exist
  const uint32_t bar0 = smem_u32(bars);
  enum { K_FULL = 0, K_EMPTY = NK, V_FULL = 2 * NK, V_EMPTY = V_FULL + NV, S_FULL = V_EMPTY + NV, P_FULL = S_FULL + SB, PV_DONE = P_FULL + SB, O_DONE = PV_DONE + SB,
         Q_FULL, Q_READ, M_READY /* [2] */, V_CLEAN = M_READY + 2, N_BARS };
  static_assert(N_BARS <= 31, "barrier slots");
  uint8_t* q_s = base + L::OFF_Q;
  auto BAR = [&](int which, int idx) { return bar0 + 8u * (uint32_t)(which + idx); };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t g = blockIdx.y, unit = blockIdx.x, p_units = p.p_splits * p.row_tiles;
  const bool shared = unit < p_units;
  uint32_t item0, n_q, split, row0, n_rows, tps;       // first item, items, split, first row in the map, the unit's rows end here, tiles per split
  if (shared) {
    split = unit / p.row_tiles;
    item0 = (unit % p.row_tiles) * p.items_per_tile;
    n_q = min(p.items_per_tile, p.n_items - item0);
    row0 = p.p_row0; n_rows = p.p_rows; tps = p.p_tps;
  } else {
    uint32_t lo = 0, hi = p.n_items - 1;
    while (lo < hi) { const uint32_t mid = (lo + hi + 1) / 2; if (unit >= p.cta0[mid]) lo = mid; else hi = mid - 1; }
    item0 = lo; n_q = 1; split = unit - p.cta0[lo];
    row0 = p.seq[lo] * p.max_seq + p.own_row0; n_rows = p.rows[lo]; tps = p.tps;
  }
  const CUtensorMap* mk = shared ? &tm_pk : &tm_k;
  const CUtensorMap* mv = shared ? &tm_pv : &tm_v;
  const bool once = !shared || p.row_tiles == 1;                       // nobody else reads the unit's rows: they need not stay in L2
  const uint32_t tiles = (n_rows + 63) / 64, tile0 = split * tps, n_tiles = min(tiles, tile0 + tps) - tile0;
  const uint32_t pairs = n_q * p.G;                                     // query rows, two lanes each
  const uint32_t live_warps = (2 * pairs + 31) / 32;                    // of each softmax group
  const bool ragged = (tile0 + n_tiles) * 64 > n_rows;                  // the last tile reaches past the unit's rows

  if (warp == 1 && lane == 0) {
    *s_err = 0;
    for (int i = 0; i < NK; ++i) { mbar_init(BAR(K_FULL, i), 1); mbar_init(BAR(K_EMPTY, i), 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(BAR(V_FULL, i), 1); mbar_init(BAR(V_EMPTY, i), 1); }
    for (int i = 0; i < SB; ++i) { mbar_init(BAR(S_FULL, i), 1); mbar_init(BAR(P_FULL, i), 32 * live_warps); mbar_init(BAR(PV_DONE, i), 1); }
    mbar_init(BAR(O_DONE, 0), 1);
    mbar_init(BAR(Q_FULL, 0), 128 * GRP);
    mbar_init(BAR(Q_READ, 0), 128 * GRP);
    mbar_init(BAR(M_READY, 0), 32 * live_warps); mbar_init(BAR(M_READY, 1), 32 * live_warps);
    mbar_init(BAR(V_CLEAN, 0), 1);
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(smem_u32((const void*)s_tmem), L::TMEM_COLS);
    tmem_relinquish();
    tc_fence_before();
  }
  if (warp == 0 && lane == 0) { prefetch_tmap(mk); prefetch_tmap(mv); }
  pdl_wait();
  pdl_trigger();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const uint32_t t_q = tmem + L::T_Q, t_s0 = tmem + L::T_S, t_o = tmem + L::T_O;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer, K ----
    if (lane == 0) {
      for (uint32_t j = 0; j < n_tiles; ++j) {
        const uint32_t st = j % NK, u = j / NK;
        if (j == 2) mbar_wait(BAR(Q_READ, 0), 0, s_err, WAIT_QFULL);         // the third slot stages query rows until then
        mbar_wait(BAR(K_EMPTY, st), (u & 1) ^ 1, s_err, WAIT_EMPTY);
        mbar_expect_tx(BAR(K_FULL, st), L::KV_BYTES);
        const uint32_t dst = smem_u32(base + L::OFF_K + st * L::KV_BYTES);
        if (once) tma_load_3d_hint(dst, mk, 0, (int)(row0 + (tile0 + j) * 64), (int)(g * CH), BAR(K_FULL, st), l2_policy_evict_first());
        else tma_load_3d(dst, mk, 0, (int)(row0 + (tile0 + j) * 64), (int)(g * CH), BAR(K_FULL, st));
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ TMA producer, V ----
    if (lane == 0) {
      for (uint32_t j = 0; j < n_tiles; ++j) {
        const uint32_t st = j % NV, u = j / NV;
        if (j == 1) mbar_wait(BAR(Q_READ, 0), 0, s_err, WAIT_QFULL);         // ... and the second V slot
        mbar_wait(BAR(V_EMPTY, st), (u & 1) ^ 1, s_err, WAIT_EMPTY);
        mbar_expect_tx(BAR(V_FULL, st), L::KV_BYTES);
        const uint32_t dst = smem_u32(base + L::OFF_V + st * L::KV_BYTES);
        if (once) tma_load_3d_hint(dst, mv, 0, (int)(row0 + (tile0 + j) * 64), (int)(g * CH), BAR(V_FULL, st), l2_policy_evict_first());
        else tma_load_3d(dst, mv, 0, (int)(row0 + (tile0 + j) * 64), (int)(g * CH), BAR(V_FULL, st));
      }
    }
    __syncwarp();
    if (ragged) {
      const uint32_t j = n_tiles - 1, st = j % NV, from = n_rows - (tile0 + j) * 64;
      mbar_wait(BAR(V_FULL, st), (j / NV) & 1, s_err, WAIT_VFULL);
      for (uint32_t i = lane; i < (64 - from) * 8 * CH; i += 32) {
        const uint32_t c = i / ((64 - from) * 8), w = i % ((64 - from) * 8);
        *reinterpret_cast<uint4*>(base + L::OFF_V + st * L::KV_BYTES + c * (64 * 128) + from * 128 + w * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(V_CLEAN, 0));
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer, scores ----
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc_qk = umma_idesc(128, 64, 0);
    uint64_t k_desc[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) k_desc[i] = smem_desc(smem_u32(base + L::OFF_K + i * L::KV_BYTES), 16, 1024);
    const uint64_t q_desc = smem_desc(smem_u32(q_s), 16, 1024);
    mbar_wait(BAR(Q_FULL, 0), 0, s_err, WAIT_QFULL);
    tc_fence_after();
    for (uint32_t j = 0; j < n_tiles; ++j) {
      const uint32_t sb = j % SB, st = j % NK;
      if (j >= (uint32_t)SB) mbar_wait(BAR(PV_DONE, sb), ((j - SB) / SB) & 1, s_err, WAIT_MMA);
      mbar_wait(BAR(K_FULL, st), (j / NK) & 1, s_err, WAIT_KFULL);
      tc_fence_after();
      const uint64_t kd = st == 0 ? k_desc[0] : (st == 1 ? k_desc[1] : k_desc[2]);
      const uint32_t ts = t_s0 + sb * 64;
      constexpr int TS_STEPS = L::TQC * 4;     // the dims whose Q chunks sit in tensor memory, then those from shared memory
#pragma unroll
      for (int ks = 0; ks < TS_STEPS; ++ks)
        umma_f16_ts(leader, ts, t_q + ks * 8, kd + (uint64_t)(((ks >> 2) * (64 * 128) + (ks & 3) * 32) >> 4), idesc_qk, ks > 0);
#pragma unroll
      for (int ks = TS_STEPS; ks < HD / 16; ++ks)
        umma_f16_ss(leader, ts, q_desc + (uint64_t)((((ks - TS_STEPS) >> 2) * (128 * 128) + (ks & 3) * 32) >> 4),
                    kd + (uint64_t)(((ks >> 2) * (64 * 128) + (ks & 3) * 32) >> 4), idesc_qk, ks > 0 ? 1u : 0u);
      umma_commit_elected(leader, BAR(K_EMPTY, st));
      umma_commit_elected(leader, BAR(S_FULL, sb));
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ MMA issuer, P V ----
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc_pv = umma_idesc(128, HD, 1);
    uint64_t v_desc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v_desc[i] = smem_desc(smem_u32(base + L::OFF_V + i * L::KV_BYTES), 64 * 128, 1024);
    for (uint32_t j = 0; j < n_tiles; ++j) {
      const uint32_t sb = j % SB, st = j % NV;
      mbar_wait(BAR(P_FULL, sb), (j / SB) & 1, s_err, WAIT_QFULL);
      mbar_wait(BAR(V_FULL, st), (j / NV) & 1, s_err, WAIT_VFULL);
      if (ragged && j == n_tiles - 1) mbar_wait(BAR(V_CLEAN, 0), 0, s_err, WAIT_VFULL);
      tc_fence_after();
      const uint64_t vd = st == 0 ? v_desc[0] : v_desc[1];
      const uint32_t tp = t_s0 + sb * 64;      // P(j): packed f16 pairs in the first 32 columns of S(j)'s tile
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        umma_f16_ts(leader, t_o, tp + ks * 8, vd + (uint64_t)((ks * 2048) >> 4), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
      umma_commit_elected(leader, BAR(V_EMPTY, st));
      umma_commit_elected(leader, BAR(PV_DONE, sb));
    }
    umma_commit_elected(leader, BAR(O_DONE, 0));
  } else {
    // ------------------------------------------------------------------ softmax + epilogue ----
    const uint32_t wg = (warp - 4) >> 2, qd = (warp - 4) & 3, row = qd * 32 + lane;
    const uint32_t lane_addr = (qd * 32) << 16;
    const bool is_lo = (row & 1u) != 0, in_use = qd < live_warps;
    const uint32_t lr = row >> 1;                      // query row: (item, head of the group)
    const bool live = lr < pairs;
    // the query rows come by cp.async into the K and the V slot that the producers leave alone until Q_READ, 32 rows each, a row's
    // 16-byte chunks XOR-swizzled against the per-row reads
    auto stage_row = [&](uint32_t pr) {
      return (pr < 32 ? base + L::OFF_K + 2 * L::KV_BYTES : base + L::OFF_V + L::KV_BYTES) + (size_t)(pr & 31u) * (HD * 4);
    };
    const uint32_t q_es = p.q_f16 ? 2u : 4u, q_ch = HD * q_es / 16, st_tid = tid - 128;
    for (uint32_t idx = st_tid; idx < pairs * q_ch; idx += 128 * GRP) {
      const uint32_t pr = idx / q_ch, c = idx % q_ch;
      const uint8_t* src = reinterpret_cast<const uint8_t*>(p.q) +
                           ((uint64_t)(item0 + pr / p.G) * p.q_col_stride + (uint64_t)(g * p.G + pr % p.G) * p.q_head_stride) * q_es + (uint64_t)c * 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(stage_row(pr) + ((c ^ (pr & 7u)) << 4))), "l"(src) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    named_bar_sync(1, 128 * GRP);
    const uint8_t* my_stage = stage_row(lr);
    auto stage_ld = [&](uint32_t c) { return *reinterpret_cast<const uint4*>(my_stage + ((c ^ (lr & 7u)) << 4)); };
    // this thread's Q row as f16 pairs, 64 dims at a time (the groups share the chunks out): high or low parts
#pragma unroll 1
    for (int c = 0; c < CH; ++c) {
      if (CH >= 2 ? (uint32_t)(c >= CH / 2) != wg : wg != 0) continue;
      uint32_t w[32];
      if (p.q_f16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 x = live && !is_lo ? stage_ld(c * 8 + i) : make_uint4(0, 0, 0, 0);      // f16 queries have no low part
          w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint4 r4 = live ? stage_ld(c * 16 + i) : make_uint4(0, 0, 0, 0);
          float4 x = *reinterpret_cast<const float4*>(&r4);
          if (is_lo) {
            x.x -= __half2float(__float2half_rn(x.x)); x.y -= __half2float(__float2half_rn(x.y));
            x.z -= __half2float(__float2half_rn(x.z)); x.w -= __half2float(__float2half_rn(x.w));
          }
          w[2 * i] = pack_h2(x.x, x.y); w[2 * i + 1] = pack_h2(x.z, x.w);
        }
      }
      if (c < L::TQC) {
        tmem_st32u(t_q + c * 32 + lane_addr, w);
      } else {
        uint8_t* dst = q_s + (c - L::TQC) * (128 * 128) + row * 128;
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(dst + ((i ^ (row & 7)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
    }
    fence_proxy_async();
    mbar_arrive(BAR(Q_READ, 0));
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(BAR(Q_FULL, 0));

    float m_st = -1.0e30f, l_sum = 0.f, m_l = m_st;
    float* sc = nullptr;                                  // where this lane's half of its row's scores goes
    if (p.scores && !shared && live)
      sc = p.scores + p.score0[item0] + ((uint64_t)g * p.G + lr) * ((n_rows + 63) & ~63u) + tile0 * 64 + (is_lo ? 32 : 0);
    if (in_use) {
      for (uint32_t j = wg; j < n_tiles; j += GRP) {
        const uint32_t b = j % SB, u = j / SB, kv0 = (tile0 + j) * 64;
        mbar_wait(BAR(S_FULL, b), u & 1, s_err, WAIT_MMA);
        tc_fence_after();
        // the two lanes of a query row share its keys out, 32 each: a lane sends the other's half of its own row (high or low
        // parts) and adds what comes back to its half
        float s[32];
        {
          float t[64];
          tmem_ld32_async(t_s0 + b * 64 + lane_addr, t);
          tmem_ld32_async(t_s0 + b * 64 + 32 + lane_addr, t + 32);
          tmem_wait_ld(t);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float give = is_lo ? t[i] : t[32 + i], keep = is_lo ? t[32 + i] : t[i];
            s[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
          }
        }
        const uint32_t key0 = kv0 + (is_lo ? 32 : 0);
        if (sc) {
          float4* d = reinterpret_cast<float4*>(sc + j * 64);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
        }
        if (kv0 + 64 > n_rows) {
#pragma unroll
          for (int i = 0; i < 32; ++i) if (key0 + i >= n_rows) s[i] = -INFINITY;
        }
        float mt = s[0];
#pragma unroll
        for (int i = 1; i < 32; ++i) mt = fmaxf(mt, s[i]);
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1)) * p.scale_log2;
        if (j > 0) {
          mbar_wait(BAR(M_READY, (j - 1) & 1), ((j - 1) >> 1) & 1, s_err, WAIT_MMA);
          m_st = s_rm[row];
        }
        float alpha = 1.f;
        bool grow = false;
        if (mt > m_st + 15.f) { alpha = ex2_approx(m_st - (mt - 7.f)); m_st = mt - 7.f; grow = true; }
        s_rm[row] = m_st;
        mbar_arrive(BAR(M_READY, j & 1));
        if (m_st != m_l) { l_sum *= ex2_approx(m_l - m_st); m_l = m_st; }
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
          const uint32_t jb = (j - 1) % SB, ju = (j - 1) / SB;
          mbar_wait(BAR(PV_DONE, jb), ju & 1, s_err, WAIT_MMA);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            float o[32];
            tmem_ld32(t_o + c * 32 + lane_addr, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(t_o + c * 32 + lane_addr, o);
          }
        }
        // weights of this lane's keys as f16 pairs, high and low parts; the even lane's row takes the high parts of all 64 keys, the odd one's the low parts
        uint32_t pw[32];
        float ls = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e0 = ex2_approx(fmaf(s[2 * i], p.scale_log2, -m_st)), e1 = ex2_approx(fmaf(s[2 * i + 1], p.scale_log2, -m_st));
          ls += e0 + e1;
          const __half2 h = __floats2half2_rn(e0, e1);
          const float2 f = __half22float2(h);
          const uint32_t hi = *reinterpret_cast<const uint32_t*>(&h), lo = pack_h2(e0 - f.x, e1 - f.y);
          const uint32_t got = __shfl_xor_sync(0xffffffffu, is_lo ? hi : lo, 1);
          pw[i] = is_lo ? got : hi;
          pw[16 + i] = is_lo ? lo : got;
        }
        l_sum += ls;
        tmem_st32u(t_s0 + b * 64 + lane_addr, pw);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(BAR(P_FULL, b));
      }
      // the row sum: the two groups' shares brought to the final reference
      mbar_wait(BAR(M_READY, (n_tiles - 1) & 1), ((n_tiles - 1) >> 1) & 1, s_err, WAIT_MMA);    // published after the last scores: the K ring is idle
      l_sum += __shfl_xor_sync(0xffffffffu, l_sum, 1);
      s_rl[wg * 128 + row] = l_sum; s_rr[wg * 128 + row] = m_l;
    }
    named_bar_sync(2, 128 * GRP);
    mbar_wait(BAR(O_DONE, 0), 0, s_err, WAIT_MMA);
    tc_fence_after();
    // ---- the records: rows to shared memory (every product has retired), whole records from there ----
    constexpr int RP = HD / 4 + 1;                       // row pitch in float4
    float4* xs = reinterpret_cast<float4*>(base + 2048);
    const uint32_t s_idx = shared ? split : p.p_splits + split;
    auto slot_of = [&](uint32_t pr) { return ((uint64_t)(item0 + pr / p.G) * p.n_heads + g * p.G + pr % p.G) * p.n_rec + s_idx; };
    if (in_use) {
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        if ((uint32_t)(c & 1) != wg) continue;           // the groups share the columns out
        float o[32];
        tmem_ld32(t_o + c * 32 + lane_addr, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] += __shfl_xor_sync(0xffffffffu, o[i], 1);
        if (live && !is_lo) {
#pragma unroll
          for (int i = 0; i < 8; ++i) xs[lr * RP + c * 8 + i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      if (live && !is_lo && wg == 0) {
        const float m = s_rm[row], l = s_rl[row] * ex2_approx(s_rr[row] - m) + s_rl[128 + row] * ex2_approx(s_rr[128 + row] - m);
        reinterpret_cast<float2*>(p.part_ml)[slot_of(lr)] = make_float2(m, l);
      }
    }
    named_bar_sync(1, 128 * GRP);
    for (uint32_t idx = st_tid; idx < pairs * (HD / 4); idx += 128 * GRP) {
      const uint32_t rr = idx / (HD / 4), c4 = idx % (HD / 4);
      reinterpret_cast<float4*>(p.part_o + slot_of(rr) * HD)[c4] = xs[rr * RP + c4];
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
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
template <int HD>
__global__ void __launch_bounds__(256, 2) pa_shared_finish_kernel(const __grid_constant__ SharedFinishParams p) {
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
  if (blockIdx.x < p.merge_ctas) {
    const uint32_t slices = HD / 4 / p.lanes, prow = blockIdx.x / slices, slice = blockIdx.x % slices, item = prow / p.n_heads, h = prow % p.n_heads;
    const uint32_t ns = p.p_splits + p.n_own[item], groups = 256 / p.lanes, grp = tid / p.lanes, ln = tid % p.lanes, dims = p.lanes * 4, d = slice * dims + tid;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + (uint64_t)prow * p.n_rec;
    const float* ob = p.part_o + (uint64_t)prow * p.n_rec * HD + slice * dims + ln * 4;
    constexpr int U = 8;
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
    const uint32_t ns = p.p_splits + p.n_own[item], rows = p.rows[item], pad = (rows + 63) & ~63u;
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

template <int HD>
static cudaError_t launch_shared_t(const SharedParams& p, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& k, const CUtensorMap& v, uint32_t n_kv,
                                   int dev, cudaStream_t st) {
  using S = ShSmem<HD>;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(pa_shared_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return e;
    attr_set[dev & 63].store(true, std::memory_order_release);
  }
  return launch_pdl(pa_shared_kernel<HD>, dim3(p.units, n_kv), dim3(S::THREADS), (size_t)S::TOTAL, st, pk, pv, k, v, p);
}
cudaError_t launch_shared(const SharedParams& p, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& k, const CUtensorMap& v, uint32_t hd, uint32_t n_kv,
                          int dev, cudaStream_t st) {
  if (hd == 256) return launch_shared_t<256>(p, pk, pv, k, v, n_kv, dev, st);
  if (hd == 128) return launch_shared_t<128>(p, pk, pv, k, v, n_kv, dev, st);
  if (hd == 64) return launch_shared_t<64>(p, pk, pv, k, v, n_kv, dev, st);
  return cudaErrorInvalidValue;
}
cudaError_t launch_shared_finish(const SharedFinishParams& p, uint32_t hd, uint32_t sum_ctas, cudaStream_t st) {
  const dim3 grid(p.merge_ctas + sum_ctas);
  if (hd == 256) return launch_pdl(pa_shared_finish_kernel<256>, grid, dim3(256), 0, st, p);
  if (hd == 128) return launch_pdl(pa_shared_finish_kernel<128>, grid, dim3(256), 0, st, p);
  if (hd == 64) return launch_pdl(pa_shared_finish_kernel<64>, grid, dim3(256), 0, st, p);
  return cudaErrorInvalidValue;
}

}  // namespace pa
