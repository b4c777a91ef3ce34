// Rotary positions of any layout and scaling (pa_rotary): q or k of any number of columns rotated from one buffer into
// another, or the front of a layer call -- q rotated, k rotated and v converted into rows of an f16 cache -- in one launch.
//
// A pair (a, b) at position p turns to m (a cos t - b sin t, b cos t + a sin t), t = p f_i.  The host keeps f_i / 2 pi in
// float64, so a thread needs one float64 product and one rint for the fraction of a turn, which goes on as an f32 pair
// (high, low): sincospif of the high part and a first-order correction by the low one leave cos and sin within 2^-23, for a
// few instructions of the slow float64 units whatever the position.  (A float64 sincos costs some two hundred.)
//
// What bounds it: HBM for prompts, latency for tokens.  A thread owns one unit of a column's heads -- two 16-byte vectors:
// the two halves of its pairs in the half layout, else two vectors of rotated or of copied dims -- and takes up to four
// columns of it at once, so that where a unit lies and what becomes of it is worked out once.  Units of rotated dims come
// first, then those that are copied, so that few warps do both.  Angles of a call whose positions the host knows are made
// ahead of the wait for the kernel before; all vectors are requested before the first is used.
#include <algorithm>

#include "pa_params.cuh"

namespace pa {

constexpr uint32_t kRotThreads = 512, kRotCols = 4;    // most threads of a CTA; columns a thread holds at once
constexpr uint32_t kRotAngles = 1024;                  // angles of a CTA's columns in shared memory

template <typename T> struct RotVec;                   // 16 bytes of T
template <> struct RotVec<__half> { static constexpr int N = 8; };
template <> struct RotVec<float> { static constexpr int N = 4; };

__device__ __forceinline__ void rot_unpack(const uint4& u, float (&v)[8], const __half*) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}
__device__ __forceinline__ void rot_unpack(const uint4& u, float (&v)[4], const float*) {
  v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
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

// where a thread's unit lies in the heads of a column, and what becomes of it
struct RotUnit {
  uint32_t head, a, b;        // its vectors (V = 1: values), elements from the head's start
  bool two, turn, halves;     // there is a second; they are rotated; as the two halves of pairs
};
template <int V>
__device__ __forceinline__ RotUnit rot_unit(uint32_t u, uint32_t heads, uint32_t hd, uint32_t n_rot, bool half) {
  RotUnit r;
  const uint32_t rv = n_rot / V, cv = (hd - n_rot) / V;               // vectors of rotated and of copied dims
  const uint32_t ru = half ? rv / 2 : (rv + 1) / 2, cu = (cv + 1) / 2;
  if (u < heads * ru) {
    const uint32_t w = u % ru;
    r.head = u / ru; r.turn = true; r.halves = half;
    r.a = w * V; r.b = r.a + (half ? n_rot / 2 : ru * V); r.two = half || r.b < n_rot;
  } else {
    u -= heads * ru;
    const uint32_t w = u % cu;
    r.head = u / cu; r.turn = r.halves = false;
    r.a = n_rot + w * V; r.b = r.a + cu * V; r.two = r.b < hd;
  }
  return r;
}
template <int V>
__host__ __device__ __forceinline__ uint32_t rot_units(uint32_t hd, uint32_t n_rot, bool half) {   // of a head
  return (half ? n_rot / V / 2 : (n_rot / V + 1) / 2) + ((hd - n_rot) / V + 1) / 2;
}

template <int N> __device__ __forceinline__ void rot_table(const float* t, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) { const float4 f = *reinterpret_cast<const float4*>(t + i); v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w; }
  } else {
    const float2 f = *reinterpret_cast<const float2*>(t);
    v[0] = f.x; v[1] = f.y;
  }
}
// neighbouring dims: V / 2 pairs
template <int V>
__device__ __forceinline__ void rot_pairs(const float* cs, const float* sn, float (&x)[V]) {
  float c[V / 2], s[V / 2];
  rot_table(cs, c); rot_table(sn, s);
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const float a = x[e], b = x[e + 1];
    x[e] = a * c[e / 2] - b * s[e / 2]; x[e + 1] = b * c[e / 2] + a * s[e / 2];
  }
}
// rotates a unit in place; cs, sn: the column's tables
template <int V>
__device__ __forceinline__ void rot_turn(const RotUnit& r, const float* cs, const float* sn, float (&x)[V], float (&y)[V]) {
  if constexpr (V == 1) {
    const uint32_t i = r.halves ? r.a : 0;
    const float c = cs[i], s = sn[i], a = x[0], b = y[0];
    x[0] = a * c - b * s; y[0] = b * c + a * s;
  } else if (r.halves) {
    float c[V], s[V];
    rot_table(cs + r.a, c); rot_table(sn + r.a, s);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = x[e], b = y[e];
      x[e] = a * c[e] - b * s[e]; y[e] = b * c[e] + a * s[e];
    }
  } else {
    rot_pairs<V>(cs + r.a / 2, sn + r.a / 2, x);
    if (r.two) rot_pairs<V>(cs + r.b / 2, sn + r.b / 2, y);
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

// V: 16-byte vectors, or 1: single values (then a unit is one pair, or two copied values), for layouts that vectors do not fit.
// Threads (units, columns); grid (column groups, unit blocks).
template <typename TI, typename TO, bool APPEND, int V>
__global__ void __launch_bounds__(kRotThreads) pa_rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) float s_c[kRotAngles], s_s[kRotAngles];
  const uint32_t tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  const uint32_t half = p.n_rot / 2, pitch = (half + 3) & ~3u, c0 = blockIdx.x * p.cpb, cols = min(p.cpb, p.n_cols - c0);
  auto angles = [&] {
    for (uint32_t i = tid; i < cols * half; i += threads) {
      const uint32_t c = i / half, k = i - c * half, col = c0 + c;
      int32_t pos;
      if (APPEND) { const uint32_t it = rot_item(p, col); pos = p.pos[it] + (int32_t)(col - p.col0[it]); }
      else pos = p.positions ? p.positions[col] : p.pos[0] + (int32_t)col;
      rot_angle(p.turns, k, pos, p.mscale, s_c[c * pitch + k], s_s[c * pitch + k]);
    }
  };
  const bool early = APPEND || !p.positions, lay = p.layout == PA_ROPE_HALF;
  if (early) angles();
  // this thread's unit: of q, of k (rotated) or of v (copied: no rotated dims)
  const uint32_t per_head = rot_units<V>(p.hd, p.n_rot, lay), uq = p.q ? p.q_heads * per_head : 0, uk = APPEND ? p.kv_heads * per_head : 0;
  const uint32_t uv = APPEND ? p.kv_heads * rot_units<V>(p.hd, 0, lay) : 0;
  uint32_t u = blockIdx.y * blockDim.x + threadIdx.x;
  const bool active = u < uq + uk + uv, is_q = !APPEND || u < uq, is_k = APPEND && !is_q && u < uq + uk;
  u = active ? u - (is_q ? 0 : is_k ? uq : uq + uk) : 0;
  RotUnit r = rot_unit<V>(u, is_q ? p.q_heads : p.kv_heads, p.hd, is_q || is_k ? p.n_rot : 0, lay);
  uint32_t pair0 = 0;
  if constexpr (V == 1)
    if (r.turn && !lay) { r.a = 2 * r.a; r.b = r.a + 1; pair0 = r.a / 2; }      // (single values: a unit of rotated dims is the pair 2i, 2i + 1)
  const TI* src = reinterpret_cast<const TI*>(is_q ? p.q : is_k ? p.k : p.v) + (is_q ? (uint64_t)r.head * p.q_head_stride : r.head * p.hd);
  const uint64_t src_cs = is_q ? p.q_col_stride : p.kv_col_stride;
  pdl_wait();
  if (APPEND) pdl_trigger();      // (y of an application may be rows that the next kernel reads at once: it starts behind this one)
  uint4 ra[kRotCols], rb[kRotCols];                    // vectors as they come (V = 1: a value in the first word)
#pragma unroll
  for (uint32_t k = 0; k < kRotCols; ++k) {
    const uint32_t c = threadIdx.y + k * blockDim.y;
    if (!active || c >= cols) continue;
    const TI* at = src + (c0 + c) * src_cs;
    if constexpr (V == 1) { ra[k].x = __float_as_uint((float)at[r.a]); if (r.two) rb[k].x = __float_as_uint((float)at[r.b]); }
    else { ra[k] = *reinterpret_cast<const uint4*>(at + r.a); if (r.two) rb[k] = *reinterpret_cast<const uint4*>(at + r.b); }
  }
  if (!early) angles();                                // positions of the device: their angles while the vectors are on their way
  __syncthreads();
#pragma unroll
  for (uint32_t k = 0; k < kRotCols; ++k) {
    const uint32_t c = threadIdx.y + k * blockDim.y;
    if (!active || c >= cols) continue;
    TO* out = nullptr;
    __half* row = nullptr;
    if (is_q) out = reinterpret_cast<TO*>(p.q_out) + (c0 + c) * p.q_out_col_stride + (uint64_t)r.head * p.q_out_head_stride;
    else {
      const uint32_t it = rot_item(p, c0 + c);
      row = (is_k ? p.k_cache : p.v_cache) + (p.row[it] + (c0 + c - p.col0[it])) * (uint64_t)(p.kv_heads * p.hd) + r.head * p.hd;
    }
    if constexpr (V > 1 && sizeof(TI) == sizeof(TO)) {
      if (is_q && !r.turn) {                           // copied as they are
        *reinterpret_cast<uint4*>(out + r.a) = ra[k];
        if (r.two) *reinterpret_cast<uint4*>(out + r.b) = rb[k];
        continue;
      }
    }
    float x[V], y[V];
    if constexpr (V == 1) { x[0] = __uint_as_float(ra[k].x); y[0] = r.two ? __uint_as_float(rb[k].x) : 0.f; }
    else {
      rot_unpack(ra[k], x, (const TI*)nullptr);
      if (r.two) rot_unpack(rb[k], y, (const TI*)nullptr);
    }
    if (r.turn) rot_turn<V>(r, s_c + c * pitch + pair0, s_s + c * pitch + pair0, x, y);
    if (is_q) {
      if constexpr (V == 1) { out[r.a] = (TO)x[0]; if (r.two) out[r.b] = (TO)y[0]; }
      else { rot_store<false>(out + r.a, x); if (r.two) rot_store<false>(out + r.b, y); }
    } else {
      if constexpr (V == 1) { row[r.a] = f16_rne(x[0]); if (r.two) row[r.b] = f16_rne(y[0]); }
      else { rot_store<true>(row + r.a, x); if (r.two) rot_store<true>(row + r.b, y); }
    }
  }
}

template <typename TI, typename TO, bool APPEND, int V>
static cudaError_t launch_rotary_v(RotaryParams p, uint32_t sms, cudaStream_t st) {
  const bool lay = p.layout == PA_ROPE_HALF;
  const uint32_t per_head = rot_units<V>(p.hd, p.n_rot, lay), units = (p.q ? p.q_heads * per_head : 0) + (APPEND ? p.kv_heads * (per_head + rot_units<V>(p.hd, 0, lay)) : 0);
  // CTAs of up to 384 units of a column, of several columns where they have few; a thread takes four columns, fewer while that
  // leaves SMs without a CTA
  const uint32_t blocks = (units + 383) / 384, x = ((units + blocks - 1) / blocks + 31) & ~31u, pitch = (p.n_rot / 2 + 3) & ~3u;
  const uint32_t y = std::max(1u, std::min(std::min(256 / x, p.n_cols), kRotAngles / pitch));
  const uint32_t k = std::max(1u, std::min(std::min(kRotCols, kRotAngles / pitch / y), (uint32_t)((uint64_t)p.n_cols * blocks / y / (2 * sms))));
  p.cpb = y * k;
  return launch_pdl(pa_rotary_kernel<TI, TO, APPEND, V>, dim3((p.n_cols + p.cpb - 1) / p.cpb, blocks), dim3(x, y), 0, st, p);
}
template <typename TI, typename TO, bool APPEND>
static cudaError_t launch_rotary_t(const RotaryParams& p, uint32_t sms, cudaStream_t st) {
  constexpr int V = RotVec<TI>::N;
  // vectors: every address a whole vector, and in the half layout both halves of the rotated dims whole vectors
  const uint32_t mo = (uint32_t)std::min<size_t>(16, V * sizeof(TO)) - 1;
  bool vec = p.n_rot % (p.layout == PA_ROPE_HALF ? 2 * V : V) == 0;
  if (p.q) vec = vec && !((uintptr_t)p.q & 15) && !((uintptr_t)p.q_out & mo) && !(p.q_col_stride % V) && !(p.q_head_stride % V) && !(p.q_out_col_stride % V) && !(p.q_out_head_stride % V);
  if (APPEND) vec = vec && !((uintptr_t)p.k & 15) && !((uintptr_t)p.v & 15) && !(p.kv_col_stride % V);
  return vec ? launch_rotary_v<TI, TO, APPEND, V>(p, sms, st) : launch_rotary_v<TI, TO, APPEND, 1>(p, sms, st);
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
