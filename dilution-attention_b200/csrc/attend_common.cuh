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

#include "lane_rows.cuh"

namespace dil {
namespace attend {

constexpr int kSpan = 64;      // tokens per entry of the document ranges

// Documents of a span of tokens.  lo, hi: smallest and largest id that is not negative (INT_MAX, -1: none);
// pure: every token of the span has the one id lo; holes: some have a negative id.
struct DocRange {
  int lo, hi, pure, holes;
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
// finite.  Values of padding (a negative id) are zeros in their tiles; a later token's or another document's are not, since rows of
// the same tile may see them.  So a kernel whose finished rows are not finite asks here whether any such value is behind it, and only
// then computes the row again, with masked pairs passed over: no cost to calls whose values are finite, little to those whose rows are
// no numbers by right, and to the rows of a tile with such a value a walk over their pairs (lane_rows.cuh).  (lse has no such products
// and stays as it is.)  B1 H4 T4096 heads of 64, forward and backward, us: finite 380; a NaN in key 0 342, in
// key 2000 2080, in all of dout 264, in query 2000 2550, in the first token's dout 4620, in a token of padding 276.

// Keys that query i may see end at key_end, queries that may see key j begin at first_query.
__device__ __forceinline__ int key_end(const Row& r, int i) { return min(r.t, max(i + 1, r.prefix)); }
__device__ __forceinline__ int first_query(const Row& r, int j) { return j < r.prefix ? 0 : j; }

// Whether a token that the row's tile has had to do with, but the row does not see, holds a value that is not finite.  Half tiles
// [h0, h1); visited(h): the tile has had to do with half tile h; bad(x): token x is such a one.
template <typename V, typename B> __device__ __forceinline__ bool masked_not_finite(int h0, int h1, V visited, B bad) {
  const int lane = threadIdx.x & 31;
  for (int h = h0; h < h1; h += 32)
    for (unsigned todo = __ballot_sync(0xffffffffu, h + lane < h1 && visited(h + lane)); todo; todo &= todo - 1) {
      const int x = (h + __ffs(todo) - 1) * 64 + lane;
      if (__any_sync(0xffffffffu, bad(x) || bad(x + 32))) return true;
    }
  return false;
}
template <typename T, int D> __device__ __forceinline__ bool finite_row(const T* p) {
  constexpr int N = 16 / (int)sizeof(T);
  float s = 0.f;
#pragma unroll 4
  for (int c = 0; c < D / N; ++c) {
    const uint4 w = reinterpret_cast<const uint4*>(p)[c];
#pragma unroll
    for (int e = 0; e < N; ++e) s = fmaf(to_f32(reinterpret_cast<const T*>(&w)[e]), 0.f, s);
  }
  return s == 0.f;
}
// Of query i, over `rows` of the keys (a tile of the tensor-core kernels; the others' are half of one).
template <typename T, int D> __device__ __forceinline__ bool masked_keys_not_finite(const Row& r, int i, const T* rows) {
  const int i0 = i & ~127;
  return masked_not_finite(r.docs != nullptr ? 0 : max(i + 1, r.prefix) / 64, (key_end(r, i0 + 127) + 63) / 64,
                           [&](int h) { return tile_visible(r, i0, i0 + 127, 64 * h, 64 * h + 63); },
                           [&](int j) { return j < r.t && !sees(r, i, j) && !finite_row<T, D>(rows + (int64_t)j * D); });
}

// What the rounding of x to T leaves off.
template <typename T> __device__ __forceinline__ float left_off(float x) { return x - to_f32(from_f32<T>(x)); }

template <typename T, int D>
__device__ __forceinline__ void redo_forward_row(const Args& a, int b, int h, int i) {
  const Row r = make_row(a, b, h);
  const int hk = h / (a.heads / a.kv_heads);
  const int64_t n = (int64_t)b * a.heads + h, nk = (int64_t)b * a.kv_heads + hk;
  const T* k = row_ptr<T>(a.k, nk, a.t, D);
  const T* v = row_ptr<T>(a.v, nk, a.t, D);
  if (!masked_keys_not_finite<T, D>(r, i, v)) return;
  LaneSums<T, D> o;
  constexpr int U = o.kSteps;
  const uint4 q = o.load(row_ptr<T>(a.q, n, a.t, D), i);
  float m = -INFINITY, s = 0.f;
  const int end = key_end(r, i);
  for (int j0 = 0; j0 < end; j0 += o.kRows) {
    bool see[U], any = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * o.R + o.own;
      see[u] = j < end && sees(r, i, j);
      any = any || see[u];
    }
    if (!__any_sync(0xffffffffu, any)) continue;
    uint4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(j0 + u * o.R + o.own, end - 1);
      x[u] = o.load(k, j);
      y[u] = o.load(v, j);
    }
    float z[U], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float dot = o.dot(q, x[u]);
      z[u] = see[u] ? score<sizeof(T) == 4>(r, dot, i, j0 + u * o.R + o.own).x : -INFINITY;
      top = fmaxf(top, z[u]);
    }
    const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m - ref);
    m = top;
    s *= f;
    o.scale(f);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (see[u]) {
        const float p = exp2f(z[u] - ref);
        s += p;
        o.add(p, y[u]);
      }
    if (o.no_number()) break;
  }
  // the groups' sums against one maximum
  const float top = o.max_over_rows(m);
  const float f = exp2f(m - (top == -INFINITY ? 0.f : top));
  s = o.over_rows(s * f);
  o.scale(f);
  o.join(s == 0.f ? 0.f : 1.f / s);
  o.store(reinterpret_cast<T*>(a.out) + (n * a.t + i) * D);
  if (a.rest != nullptr) {
#pragma unroll
    for (int e = 0; e < o.E; ++e) o.x[e] = left_off<T>(o.x[e]);
    o.store(reinterpret_cast<T*>(a.rest) + (n * a.t + i) * D);
  }
}

template <typename T, int D>
__device__ __forceinline__ void redo_dq_row(const Args& a, int b, int h, int i) {
  const Row r = make_row(a, b, h);
  const int hk = h / (a.heads / a.kv_heads);
  const int64_t n = (int64_t)b * a.heads + h, nk = (int64_t)b * a.kv_heads + hk;
  const T* k = row_ptr<T>(a.k, nk, a.t, D);
  const T* v = row_ptr<T>(a.v, nk, a.t, D);
  if (!masked_keys_not_finite<T, D>(r, i, k)) return;
  LaneSums<T, D> acc;
  constexpr int U = acc.kSteps;
  const uint4 q = acc.load(row_ptr<T>(a.q, n, a.t, D), i), g = acc.load(row_ptr<T>(a.dout, n, a.t, D), i);
  const float lse = a.lse[n * a.t + i], delta = a.delta[n * a.t + i];
  const int end = key_end(r, i);
  for (int j0 = 0; j0 < end; j0 += acc.kRows) {
    bool see[U], any = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * acc.R + acc.own;
      see[u] = j < end && sees(r, i, j);
      any = any || see[u];
    }
    if (!__any_sync(0xffffffffu, any)) continue;
    uint4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(j0 + u * acc.R + acc.own, end - 1);
      x[u] = acc.load(k, j);
      y[u] = acc.load(v, j);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float dot = acc.dot(q, x[u]), dp = acc.dot(g, y[u]);
      if (see[u]) {
        const float2 z = score<sizeof(T) == 4>(r, dot, i, j0 + u * acc.R + acc.own);
        acc.add(exp2f(z.x - lse) * (dp - delta) * z.y, x[u]);
      }
    }
    if (acc.no_number()) break;
  }
  acc.join(a.scale);
  acc.store(reinterpret_cast<T*>(a.dq) + (n * a.t + i) * D);
}

template <typename T, int D>
__device__ __forceinline__ void redo_dkv_row(const Args& a, int b, int hk, int j) {
  const int group = a.heads / a.kv_heads;
  const int64_t nk = (int64_t)b * a.kv_heads + hk;
  bool redo = false;
  for (int h = hk * group; h < (hk + 1) * group && !redo; ++h) {
    const Row r = make_row(a, b, h);
    const int64_t n = (int64_t)b * a.heads + h;
    const T* q = row_ptr<T>(a.q, n, a.t, D);
    const T* g = row_ptr<T>(a.dout, n, a.t, D);
    const int j0 = j & ~127;
    redo = masked_not_finite(
        first_query(r, j0) / 64, ((r.docs != nullptr ? a.t : j) + 63) / 64,
        [&](int x) { return tile_visible(r, 64 * x, 64 * x + 63, j0, j0 + 127); },
        [&](int i) { return i < a.t && !sees(r, i, j) && !(finite_row<T, D>(q + (int64_t)i * D) && finite_row<T, D>(g + (int64_t)i * D)); });
  }
  if (!redo) return;
  LaneSums<T, D> dk, dv;
  constexpr int U = dk.kSteps / 2;
  const uint4 k = dk.load(row_ptr<T>(a.k, nk, a.t, D), j), v = dk.load(row_ptr<T>(a.v, nk, a.t, D), j);
  bool done = false;
  for (int h = hk * group; h < (hk + 1) * group && !done; ++h) {
    const Row r = make_row(a, b, h);
    const int64_t n = (int64_t)b * a.heads + h;
    const T* q = row_ptr<T>(a.q, n, a.t, D);
    const T* g = row_ptr<T>(a.dout, n, a.t, D);
    for (int i0 = first_query(r, j); i0 < a.t && !done; i0 += dk.R * U) {
      bool see[U], any = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        see[u] = sees(r, i0 + u * dk.R + dk.own, j);
        any = any || see[u];
      }
      if (!__any_sync(0xffffffffu, any)) continue;
      uint4 x[U], y[U];
      float lse[U], delta[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * dk.R + dk.own, a.t - 1);
        x[u] = dk.load(q, i);
        y[u] = dk.load(g, i);
        lse[u] = a.lse[n * a.t + i];
        delta[u] = a.delta[n * a.t + i];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float dot = dk.dot(k, x[u]), dp = dk.dot(v, y[u]);
        if (see[u]) {
          const float2 z = score<sizeof(T) == 4>(r, dot, i0 + u * dk.R + dk.own, j);
          const float p = exp2f(z.x - lse[u]);
          dv.add(p, y[u]);
          dk.add(p * (dp - delta[u]) * z.y, x[u]);
        }
      }
      done = dk.no_number() && dv.no_number();
    }
  }
  dk.join(a.scale);
  dv.join(1.f);
  dk.store(reinterpret_cast<T*>(a.dk) + (nk * a.t + j) * D);
  dv.store(reinterpret_cast<T*>(a.dv) + (nk * a.t + j) * D);
}

// The rows first + bit of `rows`, one after the other, by a warp.  A call of its own: nothing of it may cost the kernels registers.
enum Redo { kRedoForward, kRedoDq, kRedoDkv };
template <Redo WHAT, typename T, int D> __device__ __noinline__ void redo_rows(const Args& a, int b, int h, int first, unsigned rows) {
#pragma unroll 1
  for (; rows; rows &= rows - 1) {
    const int x = first + __ffs(rows) - 1;
    if (WHAT == kRedoForward) redo_forward_row<T, D>(a, b, h, x);
    else if (WHAT == kRedoDq) redo_dq_row<T, D>(a, b, h, x);
    else redo_dkv_row<T, D>(a, b, h, x);
  }
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
  if (lane == 0) ranges[at] = DocRange{lo, hi, !neg && lo == hi, neg};
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
