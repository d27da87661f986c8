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

// Threads of a block that has a warp for each of n nodes, 8 to 16 of them.
inline int join_threads(int n) { return 32 * (n < 8 ? 8 : n > 16 ? 16 : n); }

// q, k (and v) of a head's nodes in shared memory, rows of D + 2 elements: an odd number of words.
template <int D> __device__ __forceinline__ void load_nodes(__nv_bfloat16* dst, const void* src, int64_t first, int n) {
  const uint32_t* from = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)src + first * D);
  for (int x = threadIdx.x; x < n * D / 2; x += blockDim.x)
    reinterpret_cast<uint32_t*>(dst)[x / (D / 2) * (D / 2 + 1) + x % (D / 2)] = from[x];
}
// z[nodes][nodes + 1]: scores of the nodes against the nodes that they see, -inf elsewhere.
template <int D>
__device__ __forceinline__ void node_scores(float* z, const __nv_bfloat16* q, const __nv_bfloat16* k, const Lineage& tree, const Args& a,
                                            float slope2) {
  const int n = a.nodes;
  for (int x = threadIdx.x; x < n * n; x += blockDim.x) {
    const int i = x / n, j = x % n;
    float s = -INFINITY;
    if (tree.line[i] >> j & 1) {
      s = 0.f;
#pragma unroll 8
      for (int c = 0; c < D / 2; ++c) {
        const float2 u = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(q)[i * (D / 2 + 1) + c]);
        const float2 v = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(k)[j * (D / 2 + 1) + c]);
        s = fmaf(u.x, v.x, s);
        s = fmaf(u.y, v.y, s);
      }
      s = score<true>(s, a.scale, a.cap, slope2, (float)(tree.depth[i] - tree.depth[j]));
    }
    z[i * (n + 1) + j] = s;
  }
}

// out and lse of a softmax layer's nodes.  One block per query head, a warp per node (join_threads).
// Dynamic shared memory: z [nodes][nodes + 1], then q, k, v [nodes][D + 2].
template <int D> constexpr int join_softmax_smem(int n) { return (n * (n + 1) * 4 + 15) / 16 * 16 + 3 * n * (D + 2) * 2; }
template <int D>
__global__ void __launch_bounds__(512, 2) join_softmax_kernel(Args a) {
  __shared__ Lineage tree;
  extern __shared__ __align__(16) float z[];
  const int n = a.nodes, rows = a.group * n, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(z + (n * (n + 1) + 3) / 4 * 4);
  __nv_bfloat16 *k = q + n * (D + 2), *v = k + n * (D + 2);
  const int64_t head = blockIdx.x, nk = head / a.group;
  const int h = (int)(head % ((int64_t)a.kv_heads * a.group));
  const float slope2 = a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
  load_nodes<D>(q, a.q, head * n, n);
  load_nodes<D>(k, a.kn, nk * n, n);
  load_nodes<D>(v, a.vn, nk * n, n);
  make_lineage(&tree, a.parents + nk / a.kv_heads * a.parent_stride, n);
  node_scores<D>(z, q, k, tree, a, slope2);
  __syncthreads();
  wait_for_last();                    // the chunks' parts
  constexpr int E = D / 32;
  const int warps = (int)(blockDim.x >> 5);
  auto nodes_max = [&](int x) {
    float top = -INFINITY;
    for (int y = lane; y < n; y += 32) top = fmaxf(top, z[x * (n + 1) + y]);
    return warp_max(top);
  };
  auto join_nodes = [&](int x, float from, float& s, float* o) {
    for (unsigned long long left = tree.line[x]; left; left &= left - 1) {
      const int y = __ffsll(left) - 1;
      const float p = exp2f(z[x * (n + 1) + y] - from);
      s += p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p, to_f32(v[y * (D + 2) + lane + 32 * e]), o[e]);
    }
  };
  auto store = [&](int x, float s, const float* o) {
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (head * n + x) * D + lane;
#pragma unroll
    for (int e = 0; e < E; ++e) out[32 * e] = from_f32<__nv_bfloat16>(o[e] / s);
  };
  unsigned again = 0;                 // of the warp's nodes
  for (int x = warp; x < n; x += warps) {
    const int r = (int)(head % a.group) * n + x;
    const float2* part = a.part + nk * a.chunks * rows + r;
    float top = nodes_max(x), s = 0.f, o[E];
    for (int y = lane; y < a.chunks; y += 32) top = fmaxf(top, part[(int64_t)y * rows].x);
    top = warp_max(top);
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int y0 = 0; y0 < a.chunks; y0 += 32) {
      float f = 0.f;
      if (y0 + lane < a.chunks) {
        const float2 p = part[(int64_t)(y0 + lane) * rows];
        f = exp2f(p.x - from);
        s = fmaf(p.y, f, s);
      }
      const float* src = a.pout + ((nk * a.chunks + y0) * rows + r) * D + lane;
#pragma unroll 4
      for (int y = 0; y < min(32, a.chunks - y0); ++y) {
        const float fy = __shfl_sync(0xffffffffu, f, y);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(src[(int64_t)y * rows * D + 32 * e], fy, o[e]);
      }
    }
    s = warp_sum(s);
    join_nodes(x, from, s, o);
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; ++e) bad = bad || !isfinite(o[e] / s);
    if (__any_sync(0xffffffffu, bad)) again |= 1u << x / warps;
    store(x, s, o);
    if (lane == 0) a.lse[head * n + x] = from + log2f(s);
  }
  // rows that are no numbers, over the cached keys again; behind all others, whose registers the walk does not cost there
  for (; again; again &= again - 1) {
    const int x = warp + warps * (__ffs(again) - 1), r = (int)(head % a.group) * n + x, len = cache_len(a.pos_dev, a.len, a.capacity);
    const Redone<D> got = redo_softmax<D>(a, nk, r, len + tree.depth[x], slope2, 0, len);
    const float top = fmaxf(got.m, nodes_max(x)), from = top == -INFINITY ? 0.f : top, f = exp2f(got.m - from);
    float s = got.s * f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = got.o[e] * f;
    join_nodes(x, from, s, o);
    store(x, s, o);
    // (lse stands where the values alone were no numbers)
    if (lane == 0 && !isfinite(a.lse[head * n + x])) a.lse[head * n + x] = from + log2f(s);
  }
}

// lse of a dilution layer's nodes, and their shares of the nodes' own keys: (batch * heads, nodes, nodes), 0 where a node
// does not see another.  One block per head.
template <int D>
__global__ void __launch_bounds__(512, 2) join_bids_kernel(Args a, float* __restrict__ shares) {
  __shared__ Lineage tree;
  __shared__ __nv_bfloat16 q[kMaxNodes * (D + 2)], k[kMaxNodes * (D + 2)];
  extern __shared__ float z[];                            // [nodes][nodes + 1]
  __shared__ float lse[kMaxNodes];
  const int n = a.nodes, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t nk = blockIdx.x;
  load_nodes<D>(q, a.q, nk * n, n);
  load_nodes<D>(k, a.kn, nk * n, n);
  make_lineage(&tree, a.parents + nk / a.kv_heads * a.parent_stride, n);
  let_next_in();
  node_scores<D>(z, q, k, tree, a, 0.f);
  __syncthreads();
  wait_for_last();                    // the chunks' statistics
  const int warps = (int)(blockDim.x >> 5);
  auto finish = [&](int x, float m, float s) {          // with the nodes that x sees
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
  };
  unsigned again = 0;                 // of the warp's nodes: those whose statistics are no numbers
  for (int x = warp; x < n; x += warps) {
    const float2* part = a.part + nk * a.chunks * n + x;
    float m = -INFINITY, s = 0.f;
    for (int y = lane; y < a.chunks; y += 32) m = fmaxf(m, part[(int64_t)y * n].x);
    m = warp_max(m);
    for (int y = lane; y < a.chunks; y += 32) {
      const float2 p = part[(int64_t)y * n];
      s = fmaf(p.y, exp2f(p.x - (m == -INFINITY ? 0.f : m)), s);
    }
    s = warp_sum(s);
    if (!isfinite(s) || m == INFINITY) again |= 1u << x / warps;
    finish(x, m, s);
  }
  for (; again; again &= again - 1) {
    const int x = warp + warps * (__ffs(again) - 1), len = cache_len(a.pos_dev, a.len, a.capacity);
    const float2 p = redo_stats<D>(a, nk, x, len + tree.depth[x], 0.f, 0, len);
    finish(x, p.x, p.y);
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
  wait_for_last();
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
  wait_for_last();
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
