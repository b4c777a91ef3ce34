// Rotary positions of any layout and scaling (pa_rotary): q or k of any number of columns rotated from one buffer into
// another, or the front of a layer call -- q rotated, k rotated and v converted into rows of an f16 cache -- in one launch.
//
// A pair (a, b) at position p turns to m (a cos t - b sin t, b cos t + a sin t), t = p f_i.  The host keeps f_i / 2 pi in
// float64, so a thread needs one float64 product and one rint for the fraction of a turn, which goes on as an f32 pair
// (high, low): sincospif of the high part and a first-order correction by the low one leave cos and sin within 2^-23, for a
// few instructions of the slow float64 units whatever the position.  (A float64 sincos costs some two hundred.)
//
// What bounds it: HBM for prompts, latency for tokens.  A CTA takes as many columns as give its 256 threads up to four units
// each, a unit being two 16-byte vectors (the two halves of pairs of the half layout, neighbours otherwise).  Angles of a
// call whose positions the host knows are made ahead of the wait for the kernel before; all vectors are requested before the
// first is used.
#include <algorithm>

#include "pa_params.cuh"

namespace pa {

constexpr int kRotThreads = 256, kRotUnits = 4;        // threads of a CTA, units a thread holds at once
constexpr uint32_t kRotAngles = 1024;                  // angles of a CTA's columns in shared memory

template <typename T> struct RotVec;                   // 16 bytes of T
template <> struct RotVec<__half> { static constexpr int N = 8; };
template <> struct RotVec<float> { static constexpr int N = 4; };

template <int N> __device__ __forceinline__ void rot_load(const __half* p, float (&v)[N]) {
  static_assert(N == 8, "a vector of halves");
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}
template <int N> __device__ __forceinline__ void rot_load(const float* p, float (&v)[N]) {
  static_assert(N == 4, "a vector of floats");
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
template <bool CACHE> __device__ __forceinline__ __half rot_half(float x) { return CACHE ? f16_rne(x) : __float2half_rn(x); }
template <bool CACHE, int N> __device__ __forceinline__ void rot_store(__half* p, const float (&v)[N]) {
  __half h[N];
#pragma unroll
  for (int i = 0; i < N; ++i) h[i] = rot_half<CACHE>(v[i]);
  if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
}
template <bool CACHE, int N> __device__ __forceinline__ void rot_store(float* p, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}

// one array of heads: where unit u of a column's heads lies and what becomes of it
template <int V>
struct RotUnit { uint32_t head, a, b, pair; bool half_pair, turn; };   // element offsets of its two vectors (V = 1: of its two values)

template <int V>
__device__ __forceinline__ RotUnit<V> rot_unit(uint32_t u, uint32_t hd, uint32_t n_rot, uint32_t layout, bool rotates) {
  RotUnit<V> r;
  const uint32_t per_head = hd / (2 * V), w = u % per_head;
  r.head = u / per_head;
  if (layout == PA_ROPE_HALF && rotates && w * 2 * V < n_rot) {
    r.half_pair = true; r.turn = true; r.a = w * V; r.b = n_rot / 2 + w * V; r.pair = w * V;
  } else {
    r.half_pair = false; r.a = w * 2 * V; r.b = r.a + V; r.pair = r.a / 2;
    r.turn = rotates && layout == PA_ROPE_INTERLEAVED && r.a < n_rot;
  }
  return r;
}

// rotates the 2 V values of a unit in place
template <int V>
__device__ __forceinline__ void rot_turn(const RotUnit<V>& r, uint32_t n_rot, const float* cs, const float* sn, float (&x)[V], float (&y)[V]) {
  if (!r.turn) return;
  if (r.half_pair) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float c = cs[r.pair + e], s = sn[r.pair + e], a = x[e], b = y[e];
      x[e] = a * c - b * s; y[e] = b * c + a * s;
    }
  } else if constexpr (V == 1) {
    const float c = cs[r.pair], s = sn[r.pair], a = x[0], b = y[0];
    x[0] = a * c - b * s; y[0] = b * c + a * s;
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const uint32_t i = r.pair + e / 2, j = i + V / 2;
      if (2 * i < n_rot) {
        const float c = cs[i], s = sn[i], a = x[e], b = x[e + 1];
        x[e] = a * c - b * s; x[e + 1] = b * c + a * s;
      }
      if (2 * j < n_rot) {
        const float c = cs[j], s = sn[j], a = y[e], b = y[e + 1];
        y[e] = a * c - b * s; y[e + 1] = b * c + a * s;
      }
    }
  }
}

__device__ __forceinline__ void rot_angle(const double* turns, uint32_t i, int32_t pos, float mscale, float& c, float& s) {
  double r = (double)pos * turns[i];
  r -= rint(r);
  const float hi = (float)r, d = (float)(r - (double)hi) * 6.283185307179586f;
  float c0, s0;
  sincospif(2.0f * hi, &s0, &c0);
  c = (c0 - s0 * d) * mscale;
  s = (s0 + c0 * d) * mscale;
}

// the item of a column: items own consecutive columns, col0 ascending
__device__ __forceinline__ uint32_t rot_item(const RotaryParams& p, uint32_t col) {
  if (p.one_each) return col;
  uint32_t lo = 0, hi = p.n_items - 1;
  while (lo < hi) { const uint32_t mid = (lo + hi + 1) / 2; if (col >= p.col0[mid]) lo = mid; else hi = mid - 1; }
  return lo;
}

// V: 16-byte vectors, or 1: single values, for layouts that vectors do not fit
template <typename TI, typename TO, bool APPEND, int V>
__global__ void __launch_bounds__(kRotThreads) pa_rotary_kernel(const RotaryParams p) {
  __shared__ __align__(16) float s_c[kRotAngles], s_s[kRotAngles];
  const uint32_t tid = threadIdx.x, half = p.n_rot / 2, c0 = blockIdx.x * p.cpb, cols = min(p.cpb, p.n_cols - c0);
  auto angles = [&] {
    for (uint32_t i = tid; i < cols * half; i += kRotThreads) {
      const uint32_t c = i / half, col = c0 + c;
      int32_t pos;
      if (APPEND) { const uint32_t it = rot_item(p, col); pos = p.pos[it] + (int32_t)(col - p.col0[it]); }
      else pos = p.positions ? p.positions[col] : p.pos[0] + (int32_t)col;
      rot_angle(p.turns, i % half, pos, p.mscale, s_c[i], s_s[i]);
    }
  };
  const bool early = APPEND || !p.positions;
  if (early) angles();
  pdl_wait();
  pdl_trigger();
  const uint32_t uq = p.q ? p.q_heads * (p.hd / (2 * V)) : 0, uk = APPEND ? p.kv_heads * (p.hd / (2 * V)) : 0, upc = uq + 2 * uk, total = cols * upc;
  for (uint32_t w0 = tid; w0 == tid || w0 < total; w0 += kRotThreads * kRotUnits) {
    float x[kRotUnits][V], y[kRotUnits][V];
#pragma unroll
    for (int k = 0; k < kRotUnits; ++k) {
      const uint32_t w = w0 + k * kRotThreads;
      if (w >= total) continue;
      const uint32_t col = c0 + w / upc;
      uint32_t u = w % upc;
      const TI* src;
      if (!APPEND || u < uq) {
        const RotUnit<V> r = rot_unit<V>(u, p.hd, p.n_rot, p.layout, true);
        src = reinterpret_cast<const TI*>(p.q) + (uint64_t)col * p.q_col_stride + (uint64_t)r.head * p.q_head_stride;
        if constexpr (V == 1) { x[k][0] = (float)src[r.a]; y[k][0] = (float)src[r.b]; }
        else { rot_load(src + r.a, x[k]); rot_load(src + r.b, y[k]); }
      } else {
        const bool is_k = u < uq + uk;
        u -= is_k ? uq : uq + uk;
        const RotUnit<V> r = rot_unit<V>(u, p.hd, p.n_rot, p.layout, is_k);
        src = reinterpret_cast<const TI*>(is_k ? p.k : p.v) + (uint64_t)col * p.kv_col_stride + r.head * p.hd;
        if constexpr (V == 1) { x[k][0] = (float)src[r.a]; y[k][0] = (float)src[r.b]; }
        else { rot_load(src + r.a, x[k]); rot_load(src + r.b, y[k]); }
      }
    }
    if (w0 == tid) {
      if (!early) angles();   // positions of the device: their angles while the first vectors are on their way
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kRotUnits; ++k) {
      const uint32_t w = w0 + k * kRotThreads;
      if (w >= total) continue;
      const uint32_t c = w / upc, col = c0 + c;
      uint32_t u = w % upc;
      if (!APPEND || u < uq) {
        const RotUnit<V> r = rot_unit<V>(u, p.hd, p.n_rot, p.layout, true);
        rot_turn<V>(r, p.n_rot, s_c + c * half, s_s + c * half, x[k], y[k]);
        TO* dst = reinterpret_cast<TO*>(p.q_out) + (uint64_t)col * p.q_out_col_stride + (uint64_t)r.head * p.q_out_head_stride;
        if constexpr (V == 1) { dst[r.a] = (TO)x[k][0]; dst[r.b] = (TO)y[k][0]; }
        else { rot_store<false>(dst + r.a, x[k]); rot_store<false>(dst + r.b, y[k]); }
      } else {
        const bool is_k = u < uq + uk;
        u -= is_k ? uq : uq + uk;
        const RotUnit<V> r = rot_unit<V>(u, p.hd, p.n_rot, p.layout, is_k);
        rot_turn<V>(r, p.n_rot, s_c + c * half, s_s + c * half, x[k], y[k]);
        const uint32_t it = rot_item(p, col);
        __half* dst = (is_k ? p.k_cache : p.v_cache) + (p.row[it] + (col - p.col0[it])) * (uint64_t)(p.kv_heads * p.hd) + r.head * p.hd;
        if constexpr (V == 1) { dst[r.a] = f16_rne(x[k][0]); dst[r.b] = f16_rne(y[k][0]); }
        else { rot_store<true>(dst + r.a, x[k]); rot_store<true>(dst + r.b, y[k]); }
      }
    }
  }
}

template <typename TI, typename TO, bool APPEND>
static cudaError_t launch_rotary_t(RotaryParams p, uint32_t sms, cudaStream_t st) {
  constexpr int V = RotVec<TI>::N;
  // vectors: every address a whole vector, and in the half layout both halves of the rotated dims whole vectors
  const uint32_t mo = (uint32_t)std::min<size_t>(16, V * sizeof(TO)) - 1;
  bool vec = p.layout != PA_ROPE_HALF || p.n_rot % (2 * V) == 0;
  if (p.q) vec = vec && !((uintptr_t)p.q & 15) && !((uintptr_t)p.q_out & mo) && !(p.q_col_stride % V) && !(p.q_head_stride % V) && !(p.q_out_col_stride % V) && !(p.q_out_head_stride % V);
  if (APPEND) vec = vec && !((uintptr_t)p.k & 15) && !((uintptr_t)p.v & 15) && !(p.kv_col_stride % V);
  const uint32_t upc = ((p.q ? p.q_heads : 0) + (APPEND ? 2 * p.kv_heads : 0)) * (p.hd / (vec ? 2 * V : 2));
  // columns of a CTA: four units a thread, but no fewer than four CTAs an SM while there are columns for that
  const uint32_t fit = std::max(1u, (uint32_t)(kRotThreads * kRotUnits) / upc), spread = std::max(1u, p.n_cols / (4 * sms));
  p.cpb = std::max(1u, std::min(std::min(fit, spread), kRotAngles / (p.n_rot / 2)));
  const dim3 grid((p.n_cols + p.cpb - 1) / p.cpb);
  return vec ? launch_pdl(pa_rotary_kernel<TI, TO, APPEND, V>, grid, dim3(kRotThreads), 0, st, p)
             : launch_pdl(pa_rotary_kernel<TI, TO, APPEND, 1>, grid, dim3(kRotThreads), 0, st, p);
}

template <bool APPEND>
static cudaError_t launch_rotary_a(const RotaryParams& p, uint32_t sms, cudaStream_t st) {
  if (p.in_f16) return p.out_f16 ? launch_rotary_t<__half, __half, APPEND>(p, sms, st) : launch_rotary_t<__half, float, APPEND>(p, sms, st);
  return p.out_f16 ? launch_rotary_t<float, __half, APPEND>(p, sms, st) : launch_rotary_t<float, float, APPEND>(p, sms, st);
}
cudaError_t launch_rotary(const RotaryParams& p, bool append, uint32_t sms, cudaStream_t st) {
  return append ? launch_rotary_a<true>(p, sms, st) : launch_rotary_a<false>(p, sms, st);
}

}  // namespace pa
