// What a tree step over a bf16 cache has left when the cache has been streamed (tc_tree.cuh): the chunks' parts are joined, and
// the nodes meet their own keys, of which a node sees its branch alone.  Small sums of fp32 FMAs.
#pragma once

#include "tree_common.cuh"

namespace dil {
namespace tree {

// Lane l's features l, l + 32, .. of a row.
template <int D> struct LaneRow {
  float x[D / 32];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
#pragma unroll
    for (int e = 0; e < D / 32; ++e) x[e] = to_f32(p[(threadIdx.x & 31) + 32 * e]);
  }
  __device__ __forceinline__ float dot(const LaneRow& o) const {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) s = fmaf(x[e], o.x[e], s);
    return warp_sum(s);
  }
};

// (maximum, sum) of a row over the cached keys, one warp, key by key.  For rows whose statistics came out as no number: the
// block-diagonal scores of the scan multiply zeros with what another quarter's keys hold, infinities included.
template <int D>
__device__ __noinline__ float2 redo_stats(const Args& a, int64_t nk, int r, int depth, float slope2, int len) {
  LaneRow<D> q, k;
  q.load((const __nv_bfloat16*)a.q + (nk * a.group * a.nodes + r) * D);
  float m = -INFINITY, s = 0.f;
  for (int j = 0; j < len; ++j) {
    k.load((const __nv_bfloat16*)a.kc + (nk * a.capacity + j) * D);
    const float z = score<true>(q.dot(k), a.scale, a.cap, slope2, (float)(len + depth - j)), top = fmaxf(m, z);
    const float from = top == -INFINITY ? 0.f : top;
    s = s * exp2f(m - from) + exp2f(z - from);
    m = top;
  }
  return make_float2(m, s);
}

// One block of D threads per row: out and lse of a softmax layer's node.
template <int D>
__global__ void __launch_bounds__(D) join_softmax_kernel(Args a) {
  __shared__ int up[kMaxNodes], line[kMaxNodes], count;
  __shared__ float z[kMaxNodes];
  __shared__ float again[D + 2];
  const int rows = a.group * a.nodes, c = threadIdx.x, lane = c & 31, warp = c >> 5;
  const int64_t at = blockIdx.x, nk = at / rows;
  const int r = (int)(at % rows), x = r % a.nodes, b = (int)(nk / a.kv_heads);
  if (c < a.nodes) up[c] = a.parents[b * a.parent_stride + c];
  __syncthreads();
  if (c == 0) {
    int n = 0;
    for (int y = x; y >= 0;) {
      line[n++] = y;
      const int p = up[y];
      y = p >= 0 && p < y ? p : -1;
    }
    count = n;
  }
  __syncthreads();
  const int n = count;
  const float slope2 = a.slopes != nullptr ? a.slopes[(nk % a.kv_heads) * a.group + r / a.nodes] * kLog2e : 0.f;
  {
    LaneRow<D> q, k;
    q.load((const __nv_bfloat16*)a.q + at * D);
    for (int y = warp; y < n; y += D / 32) {
      k.load((const __nv_bfloat16*)a.kn + (nk * a.nodes + line[y]) * D);
      const float s = score<true>(q.dot(k), a.scale, a.cap, slope2, (float)y);
      if (lane == 0) z[y] = s;
    }
  }
  __syncthreads();
  const float2* part = a.part + nk * a.chunks * rows + r;
  float m = -INFINITY;
  for (int y = 0; y < a.chunks; ++y) m = fmaxf(m, part[(int64_t)y * rows].x);
  for (int y = 0; y < n; ++y) m = fmaxf(m, z[y]);
  const float from = m == -INFINITY ? 0.f : m;
  float s = 0.f, o = 0.f;
  for (int y = 0; y < a.chunks; ++y) {
    const float2 p = part[(int64_t)y * rows];
    const float f = exp2f(p.x - from);
    s = fmaf(p.y, f, s);
    o = fmaf(a.pout[((nk * a.chunks + y) * rows + r) * D + c], f, o);
  }
  auto nodes = [&]() {
    for (int y = 0; y < n; ++y) {
      const float p = exp2f(z[y] - from);
      s += p;
      o = fmaf(p, to_f32(((const __nv_bfloat16*)a.vn)[(nk * a.nodes + line[y]) * D + c]), o);
    }
  };
  nodes();
  if (__syncthreads_or(!isfinite(o / s))) {
    // as in redo_stats, with the values: warp 0, key by key
    if (warp == 0) {
      const int len = cache_len(a.pos_dev, a.len, a.capacity);
      LaneRow<D> q, k, v, sum;
      q.load((const __nv_bfloat16*)a.q + at * D);
      float top = -INFINITY, mass = 0.f;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) sum.x[e] = 0.f;
      for (int j = 0; j < len; ++j) {
        k.load((const __nv_bfloat16*)a.kc + (nk * a.capacity + j) * D);
        v.load((const __nv_bfloat16*)a.vc + (nk * a.capacity + j) * D);
        const float s1 = score<true>(q.dot(k), a.scale, a.cap, slope2, (float)(len + n - 1 - j)), now = fmaxf(top, s1);
        const float base = now == -INFINITY ? 0.f : now, f = exp2f(top - base), p = exp2f(s1 - base);
        mass = mass * f + p;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) sum.x[e] = sum.x[e] * f + (p == 0.f ? 0.f : p * v.x[e]);
        top = now;
      }
#pragma unroll
      for (int e = 0; e < D / 32; ++e) again[lane + 32 * e] = sum.x[e];
      if (lane == 0) { again[D] = top; again[D + 1] = mass; }
    }
    __syncthreads();
    m = again[D];
    for (int y = 0; y < n; ++y) m = fmaxf(m, z[y]);
    const float base = m == -INFINITY ? 0.f : m, f = exp2f(again[D] - base);
    s = again[D + 1] * f;
    o = again[c] * f;
    for (int y = 0; y < n; ++y) {
      const float p = exp2f(z[y] - base);
      s += p;
      o = fmaf(p, to_f32(((const __nv_bfloat16*)a.vn)[(nk * a.nodes + line[y]) * D + c]), o);
    }
  }
  reinterpret_cast<__nv_bfloat16*>(a.out)[at * D + c] = from_f32<__nv_bfloat16>(o / s);
  if (c == 0) a.lse[at] = (m == -INFINITY ? 0.f : m) + log2f(s);
}

// lse of a dilution layer's nodes, and their shares of the nodes' own keys: (batch * heads, nodes, nodes), 0 where a node
// does not see another.  One block per head.
template <int D>
__global__ void __launch_bounds__(256) join_bids_kernel(Args a, float* __restrict__ shares) {
  constexpr int P = D + 2;                                // a row's pitch in elements: an odd number of words
  __shared__ Lineage tree;
  __shared__ __nv_bfloat16 q[kMaxNodes * P], k[kMaxNodes * P];
  extern __shared__ float z[];                            // [nodes][nodes + 1]
  __shared__ float lse[kMaxNodes];
  const int n = a.nodes, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t nk = blockIdx.x;
  for (int x = tid; x < n * D / 2; x += 256) {
    const int row = x / (D / 2), c = x % (D / 2);
    reinterpret_cast<uint32_t*>(q)[row * (P / 2) + c] = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.q + nk * n * D)[x];
    reinterpret_cast<uint32_t*>(k)[row * (P / 2) + c] = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.kn + nk * n * D)[x];
  }
  make_lineage(&tree, a.parents + nk / a.kv_heads * a.parent_stride, n);
  for (int x = tid; x < n * n; x += 256) {
    const int i = x / n, j = x % n;
    float s = -INFINITY;
    if (tree.line[i] >> j & 1) {
      s = 0.f;
      for (int c = 0; c < D / 2; ++c) {
        const float2 u = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(q)[i * (P / 2) + c]);
        const float2 v = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(k)[j * (P / 2) + c]);
        s = fmaf(u.x, v.x, s);
        s = fmaf(u.y, v.y, s);
      }
      s *= a.scale * kLog2e;
    }
    z[i * (n + 1) + j] = s;
  }
  __syncthreads();
  for (int x = warp; x < n; x += 8) {
    const float2* part = a.part + nk * a.chunks * n + x;
    float m = -INFINITY, s = 0.f;
    for (int y = lane; y < a.chunks; y += 32) m = fmaxf(m, part[(int64_t)y * n].x);
    m = warp_max(m);
    for (int y = lane; y < a.chunks; y += 32) {
      const float2 p = part[(int64_t)y * n];
      s = fmaf(p.y, exp2f(p.x - (m == -INFINITY ? 0.f : m)), s);
    }
    s = warp_sum(s);
    if (!isfinite(s) || !isfinite(m)) {
      const int len = cache_len(a.pos_dev, a.len, a.capacity);
      const float2 p = redo_stats<D>(a, nk, x, tree.depth[x], 0.f, len);
      m = p.x;
      s = p.y;
    }
    float top = m;
    for (int y = lane; y < n; y += 32) top = fmaxf(top, z[x * (n + 1) + y]);
    top = warp_max(top);
    const float from = top == -INFINITY ? 0.f : top;
    float own = 0.f;
    for (int y = lane; y < n; y += 32) own += exp2f(z[x * (n + 1) + y] - from);
    s = s * exp2f(m - from) + warp_sum(own);
    if (lane == 0) {
      lse[x] = from + log2f(s);
      a.lse[nk * n + x] = lse[x];
    }
  }
  __syncthreads();
  // a key's demand through the tree, in the nodes' order: what a node leaves stands where its score stood
  if (tid < n)
    for (int x = 0; x < n; ++x) {
      float& cell = z[x * (n + 1) + tid];
      float share = 0.f, left = 0.f;
      if (tree.line[x] >> tid & 1) {
        const int up = tree.parent[x];
        const float p = exp2f(cell - lse[x]), had = up >= 0 ? z[up * (n + 1) + tid] : 0.f;
        left = had + p;
        share = p == 0.f ? 0.f : p / (left + a.eps);
      }
      cell = left;
      shares[(nk * n + x) * n + tid] = share;
    }
}

// One block of D threads per node: out of a dilution layer's node.
template <int D>
__global__ void __launch_bounds__(D) join_dilute_kernel(Args a, const float* __restrict__ shares) {
  const int n = a.nodes, c = threadIdx.x;
  const int64_t at = blockIdx.x, nk = at / n;
  const int x = (int)(at % n);
  float s = 0.f, o = 0.f;
  for (int y = 0; y < a.chunks; ++y) {
    const int64_t p = (nk * a.chunks + y) * n + x;
    s += a.psum[p];
    o += a.pout[p * D + c];
  }
  for (int y = 0; y <= x; ++y) {
    const float w = shares[at * n + y];
    if (w == 0.f) continue;
    s += w;
    o = fmaf(w, to_f32(((const __nv_bfloat16*)a.vn)[(nk * n + y) * D + c]), o);
  }
  reinterpret_cast<__nv_bfloat16*>(a.out)[at * D + c] = from_f32<__nv_bfloat16>(o / (s + a.eps));
}

// The accepted nodes' rows behind the cache's last, and the demand of their own keys: the bids of those of them (of every
// head that shares the key head) that see it.  One block per key head, a warp per accepted key.
template <int D>
__global__ void __launch_bounds__(256) accept_nodes_kernel(Args a, Accept c) {
  __shared__ Lineage tree;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = a.group * a.nodes;
  const int64_t nk = blockIdx.x;
  const int b = (int)(nk / a.kv_heads), hk = (int)(nk % a.kv_heads), len = cache_len(a.pos_dev, a.len, a.capacity);
  make_lineage(&tree, a.parents + b * a.parent_stride, a.nodes);
  for (int x = warp; x < c.accepted && (int64_t)len + x < a.capacity; x += 8) {
    const int key = path_node(a, c, b, x);
    const int64_t src = (nk * a.nodes + key) * D, dst = (nk * a.capacity + len + x) * D;
    const uint32_t* ks = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.kn + src);
    const uint32_t* vs = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.vn + src);
    for (int e = lane; e < D / 2; e += 32) {
      reinterpret_cast<uint32_t*>((__nv_bfloat16*)c.kc + dst)[e] = ks[e];
      reinterpret_cast<uint32_t*>((__nv_bfloat16*)c.vc + dst)[e] = vs[e];
    }
    if (c.advanced == nullptr) continue;
    LaneRow<D> k, q;
    k.load((const __nv_bfloat16*)a.kn + src);
    float total = 0.f;
    for (int h = 0; h < a.group; ++h) {
      const float slope2 = a.slopes != nullptr ? a.slopes[hk * a.group + h] * kLog2e : 0.f;
      for (int y = 0; y < c.accepted; ++y) {
        const int node = path_node(a, c, b, y);
        if (!(tree.line[node] >> key & 1)) continue;
        const int64_t r = nk * rows + h * a.nodes + node;
        q.load((const __nv_bfloat16*)a.q + r * D);
        total += exp2f(score<true>(q.dot(k), a.scale, a.cap, slope2, (float)(tree.depth[node] - tree.depth[key])) - a.lse[r]);
      }
    }
    if (lane == 0) c.advanced[nk * a.capacity + len + x] = total;
  }
}

}  // namespace tree
}  // namespace dil
