// Eviction by summed attention weights (pa_evict): which rows of a (sequence, kv head) stay, and moving them together.
//
// Selection.  The rows between the first n_first and the last n_recent are ranked by their sums; the k-th largest is found
// digit by digit, 8 bits of the order-preserving integer image of the sum at a time: a histogram of the candidates' digits,
// then the digit in which the k-th lies.  Up to eight CTAs of a cluster hold the images in shared memory, so that the sums
// are read once, and add up each other's histograms; every warp owns a run of neighbouring rows, so that ranks are prefix
// sums of ballots and equal sums go to the lower rows whatever the schedule.  What bounds it: the chain of four histograms
// (some 1.5 us each) and of the ballots.
//
// Moving.  A row that stays never moves up, so a CTA that walks a column slice of the kept rows in order may read a batch
// of rows, wait for all its threads and store it: what it stores lies below everything that is still to be read.  In
// place a CTA owns 64 bytes of a head's rows (K and V by themselves) and all its rows; into another sequence nothing can
// be overwritten, CTAs share the rows out and take whole rows.  What bounds it: HBM, 4 * kv_dim bytes read and written a row.
#include <algorithm>

#include "pa_params.cuh"

namespace pa {

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32, kHistCopies = 8;

__device__ __forceinline__ uint32_t sum_order(float w) {
  if (w != w) return 0xffffffffu;                                   // NaN: above everything
  const uint32_t b = __float_as_uint(w + 0.0f);                     // -0 and 0 are equal
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

struct SelShared {
  uint32_t hist[kHistCopies][256];
  uint32_t pub[4][256];          // this CTA's histogram of each digit, read by the cluster
  uint32_t cnt[2];               // this CTA's rows above the threshold or always kept, and equal to it
  uint32_t warp_up[kSelWarps], warp_eq[kSelWarps];
  uint32_t digit, left;
  uint32_t total[256];
};

// grid (cluster, kv heads, items)
__global__ void __launch_bounds__(kSelThreads) pa_evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_key[];
  __shared__ SelShared sh;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x, nc = gridDim.x, kvh = blockIdx.y, item = blockIdx.z;
  const uint32_t n = p.rows[item];
  uint32_t* list = p.list + ((uint64_t)item * p.n_kv + kvh) * p.n_keep;
  pdl_wait();
  pdl_trigger();
  if (n <= p.n_keep) {                                              // everything stays (uniform for the cluster)
    for (uint32_t i = rank * kSelThreads + tid; i < p.n_keep; i += nc * kSelThreads) list[i] = i < n ? i : 0xffffffffu;
    return;
  }
  const uint32_t per = ((n + nc - 1) / nc + 31) & ~31u, lo = min(n, rank * per), hi = min(n, lo + per);      // this CTA's rows
  const uint32_t mid0 = p.n_first, mid1 = n - p.n_recent;           // candidates: [mid0, mid1); n > n_keep >= n_first + n_recent
  const float* sums = p.sums + ((uint64_t)p.src[item] * p.n_kv + kvh) * p.max_seq;
  uint32_t left = p.n_keep - p.n_first - p.n_recent;                // candidates to keep: fewer than there are
  for (uint32_t i = lo + tid; i < hi; i += kSelThreads) s_key[i - lo] = sum_order(sums[i]);
  uint32_t prefix = 0xffffffffu, mask = 0;
  if (left) {
    prefix = 0;
    for (int pass = 0; pass < 4; ++pass) {
      const uint32_t shift = 24 - 8 * pass;
      for (uint32_t i = tid; i < kHistCopies * 256; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
      __syncthreads();                                              // (the first time: the keys are in place too)
      for (uint32_t i0 = lo; i0 < hi; i0 += kSelThreads) {
        const uint32_t i = i0 + tid;
        const uint32_t key = i < hi ? s_key[i - lo] : 0;
        const bool in = i < hi && i >= mid0 && i < mid1 && (key & mask) == prefix;
        const uint32_t d = in ? (key >> shift) & 255u : 256u;
        const uint32_t peers = __match_any_sync(0xffffffffu, d);    // one addition for all lanes of a digit: sums share their exponents
        if (in && lane == (uint32_t)__ffs(peers) - 1) atomicAdd(&sh.hist[warp % kHistCopies][d], (uint32_t)__popc(peers));
      }
      __syncthreads();
      if (tid < 256) {
        uint32_t t = 0;
#pragma unroll
        for (int c = 0; c < kHistCopies; ++c) t += sh.hist[c][tid];
        sh.pub[pass][tid] = t;
      }
      if (nc > 1) cluster_sync(); else __syncthreads();
      if (tid < 256) {
        uint32_t t = 0;
        const uint32_t at = smem_u32(&sh.pub[pass][tid]);
        for (uint32_t c = 0; c < nc; ++c) {
          uint32_t x;
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(cluster_map(at, c)) : "memory");
          t += x;
        }
        sh.total[tid] = t;
      }
      __syncthreads();
      if (warp == 0) {                                              // from the top digit down: the one in which the k-th lies
        uint32_t own[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) { own[e] = sh.total[255 - (lane * 8 + e)]; sum += own[e]; }
        uint32_t above = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t t = __shfl_up_sync(0xffffffffu, above, o); if (lane >= (uint32_t)o) above += t; }
        above -= sum;                                               // candidates in digits above this lane's
        if (above < left && left <= above + sum) {
          uint32_t a = above;
          for (int e = 0; e < 8; ++e) {
            if (left <= a + own[e]) { sh.digit = 255 - (lane * 8 + e); sh.left = left - a; break; }
            a += own[e];
          }
        }
      }
      __syncthreads();
      prefix |= sh.digit << shift;
      mask |= 255u << shift;
      left = sh.left;
    }
  } else {
    __syncthreads();
  }
  // every candidate above `prefix` stays, and the first `left` of those equal to it
  const uint32_t run = ((hi - lo + kSelThreads - 1) / kSelThreads) * 32, w0 = min(hi, lo + warp * run), w1 = min(hi, w0 + run);     // this warp's rows
  uint32_t up = 0, eq = 0;
  for (uint32_t i0 = w0; i0 < w1; i0 += 32) {
    const uint32_t i = i0 + lane;
    const bool here = i < w1, cand = here && i >= mid0 && i < mid1;
    const uint32_t key = here ? s_key[i - lo] : 0;
    up += __popc(__ballot_sync(0xffffffffu, here && (!cand || key > prefix)));
    eq += __popc(__ballot_sync(0xffffffffu, cand && key == prefix));
  }
  if (lane == 0) { sh.warp_up[warp] = up; sh.warp_eq[warp] = eq; }
  __syncthreads();
  if (warp == 0) {
    uint32_t a = sh.warp_up[lane], b = sh.warp_eq[lane];
    const uint32_t a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= (uint32_t)o) { a += x; b += y; }
    }
    sh.warp_up[lane] = a - a0; sh.warp_eq[lane] = b - b0;
    if (lane == 31) { sh.cnt[0] = a; sh.cnt[1] = b; }
  }
  if (nc > 1) cluster_sync(); else __syncthreads();
  uint32_t up_before = sh.warp_up[warp], eq_before = sh.warp_eq[warp];
  for (uint32_t c = 0; c < rank; ++c) {
    uint32_t x, y;
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(cluster_map(smem_u32(&sh.cnt[0]), c)) : "memory");
    up_before += x; eq_before += y;
  }
  const uint32_t below = (1u << lane) - 1u;
  for (uint32_t i0 = w0; i0 < w1; i0 += 32) {
    const uint32_t i = i0 + lane;
    const bool here = i < w1, cand = here && i >= mid0 && i < mid1;
    const uint32_t key = here ? s_key[i - lo] : 0;
    const uint32_t um = __ballot_sync(0xffffffffu, here && (!cand || key > prefix)), em = __ballot_sync(0xffffffffu, cand && key == prefix);
    const uint32_t er = eq_before + __popc(em & below);             // rank among the equal ones
    const bool stays = ((um >> lane) & 1u) || (((em >> lane) & 1u) && er < left);
    if (stays) list[up_before + __popc(um & below) + min(er, left)] = i;
    up_before += __popc(um); eq_before += __popc(em);
  }
  if (nc > 1) cluster_sync();                                       // nobody leaves while its counts may be read
}

constexpr int kMoveThreads = 512, kMoveRows = 8;                    // rows a thread holds at once

// One array of rows: kept row list[i] of `from` goes to row i of `to`, i in [i0, i1), `tpr` threads (16 bytes each) a row.
// In place this is one CTA's work: what a batch stores lies below what later batches read.
__device__ __forceinline__ void move_rows(const uint8_t* from, uint8_t* to, uint64_t row_bytes, const uint32_t* list, uint32_t i0, uint32_t i1, uint32_t tpr, bool in_place) {
  const uint32_t per = kMoveThreads / tpr, r = threadIdx.x / tpr, c = threadIdx.x % tpr * 16;
  for (uint32_t b = i0; b < i1; b += per * kMoveRows) {
    uint4 x[kMoveRows];
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const uint32_t i = b + k * per + r;
      if (i < i1) x[k] = *reinterpret_cast<const uint4*>(from + (uint64_t)list[i] * row_bytes + c);
    }
    if (in_place) __syncthreads();
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const uint32_t i = b + k * per + r;
      if (i < i1) *reinterpret_cast<uint4*>(to + (uint64_t)i * row_bytes + c) = x[k];
    }
  }
}

// grid (slices or chunks of K and of V, and one CTA for the sums; kv heads; items)
__global__ void __launch_bounds__(kMoveThreads) pa_evict_move_kernel(const __grid_constant__ EvictParams p) {
  const uint32_t kvh = blockIdx.y, item = blockIdx.z, half = (gridDim.x - 1) / 2;
  const uint32_t n = min(p.rows[item], p.n_keep);                   // rows that stay
  const bool in_place = p.src[item] == p.dst[item], all = p.rows[item] <= p.n_keep;
  const uint32_t* list = p.list + ((uint64_t)item * p.n_kv + kvh) * p.n_keep;
  pdl_wait();
  if (blockIdx.x == gridDim.x - 1) {
    const float* from = p.sums + ((uint64_t)p.src[item] * p.n_kv + kvh) * p.max_seq;
    float* to = p.sums + ((uint64_t)p.dst[item] * p.n_kv + kvh) * p.max_seq;
    if (!(in_place && all)) {
      for (uint32_t b = 0; b < n; b += kMoveThreads * kMoveRows) {
        float x[kMoveRows];
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
          const uint32_t i = b + k * kMoveThreads + threadIdx.x;
          x[k] = i < n ? from[list[i]] : 0.f;
        }
        if (in_place) __syncthreads();
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
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
    if (part < p.hd / 32) move_rows(from + part * 64, to + part * 64, row_bytes, list, 0, n, 4, true);
  } else if (part < p.chunks) {
    const uint32_t per = (n + p.chunks - 1) / p.chunks;
    move_rows(from, to, row_bytes, list, min(n, part * per), min(n, part * per + per), p.hd / 8, false);
  }
}

cudaError_t launch_evict(const EvictParams& pp, uint32_t sms, int dev, cudaStream_t st) {
  EvictParams p = pp;
  uint32_t most = 0;
  bool any_in = false, any_out = false;
  for (uint32_t i = 0; i < p.n_items; ++i) {
    most = std::max(most, p.rows[i]);
    (p.src[i] == p.dst[i] ? any_in : any_out) = true;
  }
  // CTAs of a selection: 8192 rows each, eight at most (a cluster costs a barrier of a microsecond per digit)
  uint32_t nc = 1;
  while (nc < 8 && nc * 8192u < most) nc *= 2;
  const uint32_t per = ((most + nc - 1) / nc + 31) & ~31u;
  if (per > kEvictKeys) return cudaErrorInvalidValue;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(pa_evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kEvictKeys * 4));
    if (e != cudaSuccess) return e;
    attr_set[dev & 63].store(true, std::memory_order_release);
  }
  cudaError_t e = launch_pdl_cluster(pa_evict_select_kernel, dim3(nc, p.n_kv, p.n_items), dim3(kSelThreads), (size_t)std::max(per, 32u) * 4, st, nc, p);
  if (e != cudaSuccess) return e;
  // rows that go to another sequence: a CTA per 64 KB of an array, and no more than four CTAs an SM in all
  const uint32_t rows_a_cta = kMoveThreads * kMoveRows / (p.hd / 8);
  p.chunks = std::max(1u, std::min((std::min(most, p.n_keep) + rows_a_cta - 1) / rows_a_cta, 4 * sms / (2 * p.n_kv * p.n_items)));
  const uint32_t half = std::max(any_in ? p.hd / 32 : 1u, any_out ? p.chunks : 1u);
  return launch_pdl(pa_evict_move_kernel, dim3(2 * half + 1, p.n_kv, p.n_items), dim3(kMoveThreads), 0, st, p);
}

}  // namespace pa
