// Softmax attention with capped scores, a distance bias, documents and a prefix: what its kernels share.
//
//   s_ij = scale q_i . k_j;  c_ij = cap tanh(s_ij / cap)  (or s_ij);  a_ij = c_ij - slope_h |i - j|
//   query i sees key j  <=>  (j <= i  or  j < prefix_b)  and  doc_i = doc_j >= 0
//   p_ij = exp(a_ij - lse_i) over the keys that i sees;  out_i = sum_j p_ij v_j
// Scores are kept in the log2 domain (z = a log2 e), lse as log2 of the sum.  A query that sees no key has out = 0,
// lse = +inf (every p of it is 0) and no gradients.
// Backward, with delta_i = dout_i . out_i over out as it was before its rounding to bf16 (out + rest): ds is a difference of
// dout . v and delta, small next to both in a row of few keys.  In bf16, error of dq by its norm without / with rest: 6 tokens
// 0.0058 / 0.0024, 1937 tokens with a cap 0.0032 / 0.0026, and 0.0025 with out divided by the sum of its rounded P~ (the roundings
// of ds and dq alone: 0.0023).
//   dv_j = sum_i p_ij dout_i;  dc_ij = p_ij (dout_i . v_j - delta_i);  ds_ij = dc_ij (1 - (c_ij / cap)^2)
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i   (heads that share a key head: summed)
#pragma once

#include <climits>

#include "common.cuh"

namespace dil {
namespace attend {

constexpr int kSpan = 64;      // tokens per entry of the document ranges

// Documents of a span of tokens.  lo, hi: smallest and largest id that is not negative (INT_MAX, -1: none);
// pure: every token of the span has the one id lo.
struct DocRange {
  int lo, hi, pure, pad;
};

struct Args {
  const void* q;          // (batch, heads, t, d)
  const void* k;          // (batch, kv_heads, t, d)
  const void* v;
  void* out;              // (batch, heads, t, d)
  void* rest;             // bf16, like out: what its rounding left off, or null
  float* lse;             // (batch, heads, t), or null
  const void* dout;       // backward: (batch, heads, t, d)
  float* delta;           // (batch, heads, t)
  void* dq;
  void* dk;
  void* dv;
  const float* slopes;    // (heads), or null
  const int* docs;        // (batch, t), or null
  const DocRange* ranges; // (batch, ceil(t / kSpan)), with docs
  const int* prefix;      // (batch), or null
  int batch, heads, kv_heads, t;
  float scale;
  float cap;              // 0: scores as they are
};

// What a (batch, head) row needs for its scores.
struct Row {
  const int* docs;
  const DocRange* ranges;
  int prefix, t;
  float pre;              // what q . k is multiplied by: scale log2 e, or scale 2 log2 e / cap in front of the tanh
  float cap2;             // cap log2 e
  float slope2;           // slope log2 e
};

__device__ __forceinline__ Row make_row(const Args& a, int b, int h) {
  Row r;
  const int spans = (a.t + kSpan - 1) / kSpan;
  r.docs = a.docs ? a.docs + (int64_t)b * a.t : nullptr;
  r.ranges = a.docs ? a.ranges + (int64_t)b * spans : nullptr;
  r.prefix = a.prefix ? a.prefix[b] : 0;
  r.t = a.t;
  r.pre = a.cap > 0.f ? a.scale * 2.f * kLog2e / a.cap : a.scale * kLog2e;
  r.cap2 = a.cap * kLog2e;
  r.slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  return r;
}

__device__ __forceinline__ bool sees(const Row& r, int i, int j) {
  bool ok = i < r.t && j < r.t && (j <= i || j < r.prefix);
  if (r.docs != nullptr && ok) ok = r.docs[i] >= 0 && r.docs[i] == r.docs[j];
  return ok;
}

// Whether any query of [i0, i1] sees any key of [j0, j1] (may say yes where none does), and whether each sees each.
// Tiles are whole numbers of spans.
__device__ __forceinline__ bool tile_visible(const Row& r, int i0, int i1, int j0, int j1) {
  if (i0 >= r.t || j0 >= r.t || (j0 > i1 && j0 >= r.prefix)) return false;
  if (r.ranges == nullptr) return true;
  int ilo = INT_MAX, ihi = -1, jlo = INT_MAX, jhi = -1;
  for (int s = i0 / kSpan; s <= min(i1, r.t - 1) / kSpan; ++s) { ilo = min(ilo, r.ranges[s].lo); ihi = max(ihi, r.ranges[s].hi); }
  for (int s = j0 / kSpan; s <= min(j1, r.t - 1) / kSpan; ++s) { jlo = min(jlo, r.ranges[s].lo); jhi = max(jhi, r.ranges[s].hi); }
  return ihi >= jlo && jhi >= ilo;
}
__device__ __forceinline__ bool tile_full(const Row& r, int i0, int i1, int j0, int j1) {
  if (i1 >= r.t || j1 >= r.t || (j1 > i0 && j1 >= r.prefix)) return false;
  if (r.ranges == nullptr) return true;
  const int id = r.ranges[i0 / kSpan].lo;
  bool one = true;
  for (int s = i0 / kSpan; s <= i1 / kSpan; ++s) one = one && r.ranges[s].pure && r.ranges[s].lo == id;
  for (int s = j0 / kSpan; s <= j1 / kSpan; ++s) one = one && r.ranges[s].pure && r.ranges[s].lo == id;
  return one;
}

// (z, 1 - (c / cap)^2) of q . k: the score in the log2 domain and what the gradient of the capped score is multiplied by.
// EXACT: CUDA's tanhf (fp32 tensors), otherwise tanh_score.
template <bool EXACT>
__device__ __forceinline__ float2 score(const Row& r, float dot, int i, int j) {
  float z, slack = 1.f;
  if (r.cap2 > 0.f) {
    const float x = dot * r.pre * (0.5f * kLn2), u = EXACT ? tanhf(x) : tanh_score(x);
    z = r.cap2 * u;
    slack = fmaf(-u, u, 1.f);
  } else {
    z = dot * r.pre;
  }
  return make_float2(fmaf(-r.slope2, fabsf((float)(i - j)), z), slack);
}

template <typename T> __device__ __forceinline__ const T* row_ptr(const void* base, int64_t row, int t, int d) {
  return reinterpret_cast<const T*>(base) + row * t * d;
}

// ---- single rows, a warp each ------------------------------------------------------------------
// A masked pair adds 0 times a value to its row's accumulator in the tile kernels, which is NaN where that value is not
// finite (a padded token's, or a later one's).  A kernel whose finished rows are not finite computes them again here, where
// masked pairs are passed over: no cost to calls whose values are finite, some milliseconds to others.
// Lane l holds features l, l + 32, ...
template <typename T, int D> struct WarpRow {
  static constexpr int E = (D + 31) / 32;
  float x[E];
  __device__ __forceinline__ void load(const T* p, int lane) {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = lane + 32 * e < D ? to_f32(p[lane + 32 * e]) : 0.f;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
  }
  __device__ __forceinline__ void fma(float f, const WarpRow& o) {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaf(f, o.x[e], x[e]);
  }
  __device__ __forceinline__ float dot(const WarpRow& o) const {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(x[e], o.x[e], s);
    return warp_sum(s);
  }
  __device__ __forceinline__ void store(T* p, int lane, float f) const {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < D) p[lane + 32 * e] = from_f32<T>(x[e] * f);
  }
  __device__ __forceinline__ void round() {        // as the stored tensor holds it
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f32(from_f32<T>(x[e]));
  }
};

// Keys that query i may see end at key_end, queries that may see key j begin at first_query.
__device__ __forceinline__ int key_end(const Row& r, int i) { return min(r.t, max(i + 1, r.prefix)); }
__device__ __forceinline__ int first_query(const Row& r, int j) { return j < r.prefix ? 0 : j; }

// What the rounding of x to T leaves off.
template <typename T> __device__ __forceinline__ float left_off(float x) { return x - to_f32(from_f32<T>(x)); }

template <typename T, int D>
__device__ __noinline__ void redo_forward_row(const Args& a, int b, int h, int i) {
  const Row r = make_row(a, b, h);
  const int lane = threadIdx.x & 31, hk = h / (a.heads / a.kv_heads);
  const int64_t n = (int64_t)b * a.heads + h, nk = (int64_t)b * a.kv_heads + hk;
  const T* k = row_ptr<T>(a.k, nk, a.t, D);
  const T* v = row_ptr<T>(a.v, nk, a.t, D);
  WarpRow<T, D> q, o, x;
  q.load(row_ptr<T>(a.q, n, a.t, D) + (int64_t)i * D, lane);
  float m = -INFINITY, s = 0.f;
  o.zero();
  const int end = key_end(r, i);
  for (int j = 0; j < end; ++j) {
    if (!sees(r, i, j)) continue;
    x.load(k + (int64_t)j * D, lane);
    const float z = score<sizeof(T) == 4>(r, q.dot(x), i, j).x;
    const float top = fmaxf(m, z);
    const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m - ref), p = exp2f(z - ref);
    x.load(v + (int64_t)j * D, lane);
    s = fmaf(s, f, p);
#pragma unroll
    for (int e = 0; e < o.E; ++e) o.x[e] = o.x[e] * f + (p == 0.f ? 0.f : p * x.x[e]);
    m = top;
  }
  const float f = s == 0.f ? 0.f : 1.f / s;
  o.store(reinterpret_cast<T*>(a.out) + (n * a.t + i) * D, lane, f);
  if (a.rest != nullptr) {
#pragma unroll
    for (int e = 0; e < o.E; ++e) o.x[e] = left_off<T>(o.x[e] * f);
    o.store(reinterpret_cast<T*>(a.rest) + (n * a.t + i) * D, lane, 1.f);
  }
  if (a.lse != nullptr && lane == 0) a.lse[n * a.t + i] = s == 0.f ? INFINITY : m + log2f(s);
}

template <typename T, int D>
__device__ __noinline__ void redo_dq_row(const Args& a, int b, int h, int i) {
  const Row r = make_row(a, b, h);
  const int lane = threadIdx.x & 31, hk = h / (a.heads / a.kv_heads);
  const int64_t n = (int64_t)b * a.heads + h, nk = (int64_t)b * a.kv_heads + hk;
  const T* k = row_ptr<T>(a.k, nk, a.t, D);
  const T* v = row_ptr<T>(a.v, nk, a.t, D);
  WarpRow<T, D> q, g, acc, x;
  q.load(row_ptr<T>(a.q, n, a.t, D) + (int64_t)i * D, lane);
  g.load(row_ptr<T>(a.dout, n, a.t, D) + (int64_t)i * D, lane);
  acc.zero();
  const float lse = a.lse[n * a.t + i], delta = a.delta[n * a.t + i];
  const int end = key_end(r, i);
  for (int j = 0; j < end; ++j) {
    if (!sees(r, i, j)) continue;
    x.load(v + (int64_t)j * D, lane);
    const float dp = g.dot(x);
    x.load(k + (int64_t)j * D, lane);
    const float2 z = score<sizeof(T) == 4>(r, q.dot(x), i, j);
    const float p = exp2f(z.x - lse);
    if (p != 0.f) acc.fma(p * (dp - delta) * z.y, x);
  }
  acc.store(reinterpret_cast<T*>(a.dq) + (n * a.t + i) * D, lane, a.scale);
}

template <typename T, int D>
__device__ __noinline__ void redo_dkv_row(const Args& a, int b, int hk, int j) {
  const int lane = threadIdx.x & 31, group = a.heads / a.kv_heads;
  const int64_t nk = (int64_t)b * a.kv_heads + hk;
  WarpRow<T, D> k, v, dk, dv, q, g;
  k.load(row_ptr<T>(a.k, nk, a.t, D) + (int64_t)j * D, lane);
  v.load(row_ptr<T>(a.v, nk, a.t, D) + (int64_t)j * D, lane);
  dk.zero();
  dv.zero();
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const Row r = make_row(a, b, h);
    const int64_t n = (int64_t)b * a.heads + h;
    for (int i = first_query(r, j); i < a.t; ++i) {
      if (!sees(r, i, j)) continue;
      q.load(row_ptr<T>(a.q, n, a.t, D) + (int64_t)i * D, lane);
      g.load(row_ptr<T>(a.dout, n, a.t, D) + (int64_t)i * D, lane);
      const float2 z = score<sizeof(T) == 4>(r, q.dot(k), i, j);
      const float p = exp2f(z.x - a.lse[n * a.t + i]), dp = g.dot(v);
      if (p == 0.f) continue;
      dv.fma(p, g);
      dk.fma(p * (dp - a.delta[n * a.t + i]) * z.y, q);
    }
  }
  dk.store(reinterpret_cast<T*>(a.dk) + (nk * a.t + j) * D, lane, a.scale);
  dv.store(reinterpret_cast<T*>(a.dv) + (nk * a.t + j) * D, lane, 1.f);
}

// ---- what runs in front of the passes ----------------------------------------------------------
// One warp per span of a sequence's document ids.
__global__ void __launch_bounds__(256) doc_ranges_kernel(const int* __restrict__ docs, int batch, int t,
                                                         DocRange* __restrict__ ranges) {
  const int spans = (t + kSpan - 1) / kSpan, lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= (int64_t)batch * spans) return;
  const int b = (int)(at / spans), i0 = (int)(at % spans) * kSpan;
  int lo = INT_MAX, hi = -1;
  bool neg = false;
  for (int i = i0 + lane; i < min(t, i0 + kSpan); i += 32) {
    const int id = docs[(int64_t)b * t + i];
    if (id < 0) neg = true;
    else { lo = min(lo, id); hi = max(hi, id); }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  neg = __any_sync(0xffffffffu, neg);
  if (lane == 0) ranges[at] = DocRange{lo, hi, !neg && lo == hi, 0};
}

// dout . (out + rest) of 16 bytes of each, in 32 bits.  (An out beyond bf16's range has no rest: inf - inf.)
template <typename T> __device__ __forceinline__ float delta_part(const Args& a, int64_t at) {
  constexpr int E = 16 / sizeof(T);
  const uint4 x = reinterpret_cast<const uint4*>(a.dout)[at], y = reinterpret_cast<const uint4*>(a.out)[at];
  const uint4 z = a.rest ? reinterpret_cast<const uint4*>(a.rest)[at] : make_uint4(0, 0, 0, 0);
  const T *g = reinterpret_cast<const T*>(&x), *o = reinterpret_cast<const T*>(&y), *r = reinterpret_cast<const T*>(&z);
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float low = to_f32(r[e]);
    s = fmaf(to_f32(g[e]), to_f32(o[e]) + (isfinite(low) ? low : 0.f), s);
  }
  return s;
}

// delta_i of every query; D / 8 (bf16) or D / 4 (fp32) lanes a row, 16 bytes each.
template <typename T, int D>
__global__ void __launch_bounds__(256) delta_kernel(Args a, int64_t rows) {
  constexpr int L = D * (int)sizeof(T) / 16;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / L;
  float s = row < rows ? delta_part<T>(a, at) : 0.f;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (row < rows && at % L == 0) a.delta[row] = s;
}

}  // namespace attend
}  // namespace dil
