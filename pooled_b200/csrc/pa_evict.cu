// Eviction by summed attention weights (pa_evict): which rows of a (sequence, kv head) stay, and moving them together.
//
// Selection.  The rows between the first n_first and the last n_recent are ranked by their sums; the k-th largest is found
// digit by digit, 8 bits of the order-preserving integer image of the sum at a time: a histogram of the candidates' digits,
// then the digit in which the k-th lies (one warp's work: done by all of them for themselves it took 0.7 us longer).  The images are in shared memory, so the sums are
// read once: of one CTA up to kEvictAlone rows, beyond of the eight of a cluster, which add up each other's histograms.  Every
// warp owns a run of neighbouring rows, so that ranks are prefix sums of ballots and equal sums go to the lower rows whatever
// the schedule.  What bounds it: the chain of four digits, 0.8 us each in one CTA, 1.6 us in a cluster (4 x 32768 rows:
// selection 13 us, move 9).
//
// Moving.  A row that stays never moves up, so a CTA that walks a column slice of the kept rows in order may read a batch
// of rows, wait for all its threads and store it: what it stores lies below everything that is still to be read.  In place a
// CTA owns 64 bytes of a head's rows, of K or of V, and all of its rows; into another sequence nothing can be overwritten, and
// CTAs share the rows out and take whole ones.  What bounds it into another sequence: HBM, 4 * kv_dim bytes a row read and written (4 x 32768 ->
// 30000 rows, 8 heads of 128: 187 us with the selection, 152 of them bytes).  In place 2 * hd / 32 CTAs a head work, a chain of batches of 512
// rows with a load and a barrier each: latency, until there are heads and sequences enough (the same 215 us; one sequence 113 us for 65,
// with 24 % of DRAM's rate; 32768 -> 4096 rows of 2 heads of 256 23 us for 16).
#include <algorithm>

#include "pa_params.cuh"

namespace pa {

constexpr int kKeys = 8, kEvictThreads = 512, kEvictWarps = kEvictThreads / 32, kEvictCtas = 8;

__device__ __forceinline__ uint32_t sum_order(float w) {
  if (w != w) return 0xffffffffu;                                   // NaN: above everything
  const uint32_t b = __float_as_uint(w + 0.0f);                     // -0 and 0 are equal
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

struct EvictShared {
  uint32_t hist[4][256];         // the candidates' digits from the highest (255) down, a histogram for each of the four
  uint32_t total[256];           // ... of the cluster
  uint32_t digit, left;          // of the k-th row: its digit, its rank among those that have it
  uint32_t cnt[2];               // this CTA's rows above the threshold or always kept, and equal to it
  uint32_t warp_up[kEvictWarps], warp_eq[kEvictWarps];
};

// grid (1, or a cluster of 8 that shares the rows out; kv heads; items)
template <bool SPLIT>
__global__ void __launch_bounds__(kEvictThreads) pa_evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_key[];
  __shared__ __align__(16) EvictShared sh;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = SPLIT ? blockIdx.x : 0, kvh = blockIdx.y, item = blockIdx.z;
  const uint32_t rows = p.rows[item];
  uint32_t* list = p.list + ((uint64_t)item * p.n_kv + kvh) * p.n_keep;
  if (tid < 256) { sh.hist[0][tid] = 0; sh.hist[1][tid] = 0; sh.hist[2][tid] = 0; sh.hist[3][tid] = 0; }
  pdl_wait();
  pdl_trigger();
  if (rows <= p.n_keep) {                                           // everything stays (the same for the whole cluster)
    for (uint32_t i = rank * kEvictThreads + tid; i < p.n_keep; i += gridDim.x * kEvictThreads) list[i] = i < rows ? i : 0xffffffffu;
    return;
  }
  const float* sums = p.sums + ((uint64_t)p.src[item] * p.n_kv + kvh) * p.max_seq;
  const uint32_t per = SPLIT ? ((rows + kEvictCtas - 1) / kEvictCtas + 31) & ~31u : rows;
  const uint32_t lo = SPLIT ? min(rows, rank * per) : 0, hi = min(rows, lo + per);        // this CTA's rows
  const uint32_t mid0 = p.n_first, mid1 = rows - p.n_recent;        // candidates: [mid0, mid1); rows > n_keep >= n_first + n_recent
  uint32_t left = p.n_keep - p.n_first - p.n_recent;                // candidates to keep: fewer than there are
  uint32_t prefix = left ? 0 : 0xffffffffu, mask = 0;
  __syncthreads();                                                  // the histograms are zero
  if (left) {
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
      const uint32_t shift = 24 - 8 * pass;
      for (uint32_t i0 = lo; i0 < hi; i0 += kEvictThreads * kKeys) {
        uint32_t key[kKeys];                                        // several at once: each would wait for its own memory round trip
        if (pass == 0) {
          float w[kKeys];
#pragma unroll
          for (int k = 0; k < kKeys; ++k) { const uint32_t i = i0 + k * kEvictThreads + tid; w[k] = i < hi ? sums[i] : 0.f; }
#pragma unroll
          for (int k = 0; k < kKeys; ++k) { const uint32_t i = i0 + k * kEvictThreads + tid; key[k] = sum_order(w[k]); if (i < hi) s_key[i - lo] = key[k]; }
        } else {
#pragma unroll
          for (int k = 0; k < kKeys; ++k) { const uint32_t i = i0 + k * kEvictThreads + tid; key[k] = i < hi ? s_key[i - lo] : 0; }
        }
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const uint32_t i = i0 + k * kEvictThreads + tid;
          if (i0 + k * kEvictThreads >= hi) break;                  // (the same for all threads)
          const bool in = i < hi && i >= mid0 && i < mid1 && (key[k] & mask) == prefix;
          const uint32_t d = 255 - ((key[k] >> shift) & 255u);
          if (pass == 0) {                                          // sign and exponent, a few values only: one addition for all lanes that have it
            const uint32_t peers = __match_any_sync(0xffffffffu, in ? d : 256u);
            if (in && lane == (uint32_t)__ffs(peers) - 1) atomicAdd(&sh.hist[0][d], (uint32_t)__popc(peers));
          } else if (in) {
            atomicAdd(&sh.hist[pass][d], 1u);
          }
        }
      }
      const uint32_t* bins = sh.hist[pass];
      if constexpr (SPLIT) {
        cluster_sync();
        if (tid < 256) {
          uint32_t t = 0;
          const uint32_t at = smem_u32(&sh.hist[pass][tid]);
#pragma unroll
          for (uint32_t c = 0; c < kEvictCtas; ++c) {
            uint32_t x;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(cluster_map(at, c)) : "memory");
            t += x;
          }
          sh.total[tid] = t;                                        // (the last digit's readers are behind the cluster's barrier)
        }
        bins = sh.total;
      }
      __syncthreads();
      // from the highest digit down: the one in which the k-th lies, eight digits a lane
      if (warp == 0) {
        const uint4 a = reinterpret_cast<const uint4*>(bins)[lane * 2], b = reinterpret_cast<const uint4*>(bins)[lane * 2 + 1];
        const uint32_t own[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        const uint32_t sum = a.x + a.y + a.z + a.w + b.x + b.y + b.z + b.w;
        uint32_t above = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t t = __shfl_up_sync(0xffffffffu, above, o); if (lane >= (uint32_t)o) above += t; }
        above -= sum;                                               // candidates in digits above this lane's
        if (above < left && left <= above + sum) {
          uint32_t rest = left - above, e = 0;
#pragma unroll
          for (int k = 0; k < 7; ++k)
            if (e == (uint32_t)k && rest > own[k]) { rest -= own[k]; e = k + 1; }
          sh.digit = 255 - (lane * 8 + e); sh.left = rest;
        }
      }
      __syncthreads();
      prefix |= sh.digit << shift;
      left = sh.left;
      mask |= 255u << shift;
    }
  } else {
    for (uint32_t i = lo + tid; i < hi; i += kEvictThreads) s_key[i - lo] = 0;            // no candidate stays, whatever its sum
    __syncthreads();
  }
  // every candidate above `prefix` stays, and the first `left` of those equal to it
  const uint32_t run = ((hi - lo + kEvictThreads - 1) / kEvictThreads) * 32, w0 = min(hi, lo + warp * run), w1 = min(hi, w0 + run);     // this warp's rows
  uint32_t up = 0, eq = 0, um_kept = 0, em_kept = 0;                // (lane t keeps the ballots of the warp's rows 32 t .. 32 t + 31)
  auto ballots = [&](uint32_t i0, uint32_t& um, uint32_t& em) {
    const uint32_t i = i0 + lane;
    const bool here = i < w1, cand = here && i >= mid0 && i < mid1;
    const uint32_t key = here ? s_key[i - lo] : 0;
    um = __ballot_sync(0xffffffffu, here && (!cand || key > prefix));
    em = __ballot_sync(0xffffffffu, cand && key == prefix);
  };
  for (uint32_t i0 = w0, t = 0; i0 < w1; i0 += 32, ++t) {
    uint32_t um, em;
    ballots(i0, um, em);
    if (lane == t) { um_kept = um; em_kept = em; }
    up += __popc(um); eq += __popc(em);
  }
  if (lane == 0) { sh.warp_up[warp] = up; sh.warp_eq[warp] = eq; }
  __syncthreads();
  uint32_t up_before = lane < warp ? sh.warp_up[lane] : 0, eq_before = lane < warp ? sh.warp_eq[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { up_before += __shfl_xor_sync(0xffffffffu, up_before, o); eq_before += __shfl_xor_sync(0xffffffffu, eq_before, o); }
  if constexpr (SPLIT) {
    if (warp == kEvictWarps - 1 && lane == 0) { sh.cnt[0] = up_before + up; sh.cnt[1] = eq_before + eq; }
    cluster_sync();
    for (uint32_t c = 0; c < rank; ++c) {
      uint32_t x, y;
      asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(cluster_map(smem_u32(&sh.cnt[0]), c)) : "memory");
      up_before += x; eq_before += y;
    }
  }
  const uint32_t below = (1u << lane) - 1u;
  for (uint32_t i0 = w0, t = 0; i0 < w1; i0 += 32, ++t) {
    uint32_t um, em;
    if (t < 32) { um = __shfl_sync(0xffffffffu, um_kept, t); em = __shfl_sync(0xffffffffu, em_kept, t); }
    else ballots(i0, um, em);
    const uint32_t er = eq_before + __popc(em & below);             // rank among the equal ones
    const bool stays = ((um >> lane) & 1u) || (((em >> lane) & 1u) && er < left);
    if (stays) list[up_before + __popc(um & below) + min(er, left)] = i0 + lane;
    up_before += __popc(um); eq_before += __popc(em);
  }
  if constexpr (SPLIT) cluster_sync();                              // nobody leaves while its counts may be read
}

constexpr int kMoveThreads = 512, kMoveRows = 8, kSumBatch = 8;

// One array of rows: kept row list[i] of `from` goes to row i of `to`, i in [i0, i1), `tpr` threads (16 bytes each) a row, ROWS rows
// a thread at once.  IN_PLACE, one CTA's work: what a batch stores lies below what later batches read, so the next one is
// requested before this one is stored.
template <int ROWS, bool IN_PLACE>
__device__ __forceinline__ void move_rows(const uint8_t* from, uint8_t* to, uint64_t row_bytes, const uint32_t* list, uint32_t i0, uint32_t i1, uint32_t tpr) {
  const uint32_t per = kMoveThreads / tpr, r = threadIdx.x / tpr, c = threadIdx.x % tpr * 16;
  uint4 x[ROWS];
  auto load = [&](uint32_t b) {
    uint32_t at[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) at[k] = b + k * per + r < i1 ? list[b + k * per + r] : 0;
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (b + k * per + r < i1) x[k] = *reinterpret_cast<const uint4*>(from + (uint64_t)at[k] * row_bytes + c);
  };
  if (IN_PLACE) load(i0);
  for (uint32_t b = i0; b < i1; b += per * ROWS) {
    if (!IN_PLACE) load(b);
    uint4 y[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) y[k] = x[k];
    if (IN_PLACE) {
      __syncthreads();
      load(b + per * ROWS);
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const uint32_t i = b + k * per + r;
      if (i < i1) *reinterpret_cast<uint4*>(to + (uint64_t)i * row_bytes + c) = y[k];
    }
  }
}

// grid (slices or chunks of K and of V, and one CTA for the sums; kv heads; items)
__global__ void __launch_bounds__(kMoveThreads, 2) pa_evict_move_kernel(const __grid_constant__ EvictParams p) {
  const uint32_t kvh = blockIdx.y, item = blockIdx.z, half = (gridDim.x - 1) / 2;
  const uint32_t n = min(p.rows[item], p.n_keep);                   // rows that stay
  const bool in_place = p.src[item] == p.dst[item], all = p.rows[item] <= p.n_keep;
  const uint32_t* list = p.list + ((uint64_t)item * p.n_kv + kvh) * p.n_keep;
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == gridDim.x - 1) {
    const float* from = p.sums + ((uint64_t)p.src[item] * p.n_kv + kvh) * p.max_seq;
    float* to = p.sums + ((uint64_t)p.dst[item] * p.n_kv + kvh) * p.max_seq;
    if (!(in_place && all)) {
      for (uint32_t b = 0; b < n; b += kMoveThreads * kSumBatch) {
        float x[kSumBatch];
#pragma unroll
        for (int k = 0; k < kSumBatch; ++k) {
          const uint32_t i = b + k * kMoveThreads + threadIdx.x;
          x[k] = i < n ? from[list[i]] : 0.f;
        }
        if (in_place) __syncthreads();
#pragma unroll
        for (int k = 0; k < kSumBatch; ++k) {
          const uint32_t i = b + k * kMoveThreads + threadIdx.x;
          if (i < n) to[i] = x[k];
        }
      }
    }
    for (uint32_t i = n + threadIdx.x; i < p.max_seq; i += kMoveThreads) to[i] = 0.f;      // (in place: rows at or past n are no longer read)
    return;
  }
  if (in_place && all) return;
  const uint32_t which = blockIdx.x / half, part = blockIdx.x % half;
  const uint64_t row_bytes = (uint64_t)p.n_kv * p.hd * 2;
  uint8_t* cache = reinterpret_cast<uint8_t*>(which ? p.v : p.k);
  const uint8_t* from = cache + (uint64_t)p.src[item] * p.max_seq * row_bytes + kvh * p.hd * 2;
  uint8_t* to = cache + (uint64_t)p.dst[item] * p.max_seq * row_bytes + kvh * p.hd * 2;
  if (in_place) {
    if (part < p.hd / 32) move_rows<kMoveRows / 2, true>(from + part * 64, to + part * 64, row_bytes, list, 0, n, 4);
  } else if (part < p.chunks) {
    const uint32_t per = (n + p.chunks - 1) / p.chunks;
    move_rows<kMoveRows, false>(from, to, row_bytes, list, min(n, part * per), min(n, part * per + per), p.hd / 8);
  }
}

cudaError_t launch_evict(const EvictParams& pp, uint32_t sms, int dev, cudaStream_t st) {
  EvictParams p = pp;
  uint32_t most = 1;
  bool any_in = false, any_out = false;
  for (uint32_t i = 0; i < p.n_items; ++i) {
    most = std::max(most, p.rows[i]);
    (p.src[i] == p.dst[i] ? any_in : any_out) = true;
  }
  const bool split = most > kEvictAlone;
  const uint32_t keys = split ? ((most + kEvictCtas - 1) / kEvictCtas + 31) & ~31u : most;
  if (keys > kEvictKeys) return cudaErrorInvalidValue;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(pa_evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kEvictKeys * 4));
    if (e != cudaSuccess) return e;
    attr_set[dev & 63].store(true, std::memory_order_release);
  }
  cudaError_t e = split ? launch_pdl_cluster(pa_evict_select_kernel<true>, dim3(kEvictCtas, p.n_kv, p.n_items), dim3(kEvictThreads), (size_t)keys * 4, st, kEvictCtas, p)
                        : launch_pdl(pa_evict_select_kernel<false>, dim3(1, p.n_kv, p.n_items), dim3(kEvictThreads), (size_t)keys * 4, st, p);
  if (e != cudaSuccess) return e;
  // rows that go to another sequence: a CTA per 64 KB of an array, and no more than four CTAs an SM in all
  const uint32_t rows_a_cta = kMoveThreads * kMoveRows / (p.hd / 8);
  p.chunks = std::max(1u, std::min((std::min(most, p.n_keep) + rows_a_cta - 1) / rows_a_cta, 4 * sms / (2 * p.n_kv * p.n_items)));
  const uint32_t half = std::max(any_in ? p.hd / 32 : 1u, any_out ? p.chunks : 1u);
  return launch_pdl(pa_evict_move_kernel, dim3(2 * half + 1, p.n_kv, p.n_items), dim3(kMoveThreads), 0, st, p);
}

}  // namespace pa
