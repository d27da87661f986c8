// Drafted tokens over a cache: what the kernels of tree steps share.
//
// A tree of N <= 64 drafted nodes continues a cache of `len` keys.  Node x sees the cached keys, its ancestors and itself;
// it stands at position len + depth(x).  A key head's rows are the nodes of the `group` query heads that share it:
// row r is node r % N of head r / N.  Keys are numbered [0, len) in the cache and len + x for node x.
#pragma once

#include "lane_rows.cuh"

namespace dil {
namespace tree {

constexpr int kMaxNodes = 64;

struct Args {
  const void* q;           // (batch, kv_heads, group, nodes, d): heads in order
  const void* kn;          // (batch, kv_heads, nodes, d)
  const void* vn;
  const void* kc;          // (batch, kv_heads, capacity, d)
  const void* vc;
  const int* parents;      // (batch or 1, nodes)
  int64_t parent_stride;   // nodes, or 0 for one tree
  const float* slopes;     // (kv_heads * group), or null
  const int* pos_dev;      // the cache's length on the device, or null
  const float* committed;  // (batch, kv_heads, capacity): the demand of a dilution layer's keys
  float* lse;              // (batch, heads, nodes): log2 of the sum of 2^z
  void* out;               // (batch, heads, nodes, d)
  float2* part;            // scratch: (batch * kv_heads, chunks, rows) (maximum, sum)
  float* pout;             // scratch: (batch * kv_heads, chunks, rows, d)
  float* psum;             // scratch: (batch * kv_heads, chunks, rows) sums of shares
  int64_t capacity;
  int len, batch, kv_heads, group, nodes, chunks;
  float scale, cap, eps;
};

// Ancestors (and the node itself) as bits, depths and checked parents of one tree.
struct Lineage {
  unsigned long long line[kMaxNodes];
  int depth[kMaxNodes], parent[kMaxNodes];
};

__device__ __forceinline__ int cache_len(const int* pos_dev, int len, int64_t capacity) {
  return pos_dev != nullptr ? (int)min((int64_t)max(*pos_dev, 0), capacity) : len;
}

// Every thread of the block calls this; a parent that is no earlier node counts as none.  Bits and depths by pointer
// doubling: six rounds, whatever the tree's depth.
__device__ __forceinline__ void make_lineage(Lineage* s, const int* parents, int nodes) {
  const int x = threadIdx.x;
  unsigned long long line = 0;
  int up = -1;
  if (x < kMaxNodes) {
    if (x < nodes) {
      up = parents[x];
      if (up < 0 || up >= x) up = -1;
      line = 1ull << x;
    }
    s->parent[x] = s->depth[x] = up;
    s->line[x] = line;
  }
  __syncthreads();
  for (int round = 0; round < 6; ++round) {
    if (x < kMaxNodes && up >= 0) {
      line |= s->line[up];
      up = s->depth[up];
    }
    __syncthreads();
    if (x < kMaxNodes) {
      s->line[x] = line;
      s->depth[x] = up;
    }
    __syncthreads();
  }
  if (x < kMaxNodes) s->depth[x] = x < nodes ? __popcll(line) - 1 : 0;
  __syncthreads();
}

// Keys of chunk c of `chunks`, whole tiles of `tile` each.
__device__ __forceinline__ int2 chunk_keys(int keys, int chunks, int c, int tile) {
  const int per = ((keys + tile - 1) / tile + chunks - 1) / chunks * tile;
  return make_int2(min(keys, c * per), min(keys, (c + 1) * per));
}

// The score of q . k in the log2 domain; far: the distance.
template <bool EXACT>
__device__ __forceinline__ float score(float dot, float scale, float cap, float slope2, float far) {
  float z;
  if (cap > 0.f)
    z = cap * kLog2e * (EXACT ? tanhf(dot * scale / cap) : tanh_score(dot * (scale / cap)));
  else
    z = dot * (scale * kLog2e);
  return fmaf(-slope2, far, z);
}

// A row that came out as no number, of a bf16 cache on the tensor cores: the block-diagonal scores of a scan multiply zeros with what
// another quarter's keys hold, and its zero weights another quarter's values, infinities included.  These walk over the cached keys
// [j0, j1) again, one warp a row (lane_rows.cuh), and end where nothing is a number any more.  Row r of key head nk, at position `at`.
// 8 heads of 64, 12 nodes over 16384 keys, us: softmax step 53, with the last key or value infinite or NaN 1410, with the first key NaN
// 54; dilution step 59, 930 and 59.
template <int D> __device__ __noinline__ float2 redo_stats(const Args& a, int64_t nk, int r, int at, float slope2, int j0, int j1) {
  using L = Lanes<__nv_bfloat16, D>;
  const L l;
  constexpr int U = 2 * L::kSteps;
  const __nv_bfloat16* k = (const __nv_bfloat16*)a.kc + nk * a.capacity * D;
  const uint4 q = l.load((const __nv_bfloat16*)a.q + (nk * a.group * a.nodes + r) * D, 0);
  float m = -INFINITY, s = 0.f;
  for (int j = j0; j < j1; j += U * L::R) {
    uint4 x[U];
    float z[U], top = m, sum = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = l.load(k, min(j + u * L::R + l.own, j1 - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j + u * L::R + l.own;
      const float dot = l.dot(q, x[u]);
      z[u] = key < j1 ? score<true>(dot, a.scale, a.cap, slope2, (float)(at - key)) : -INFINITY;
      top = fmaxf(top, z[u]);
    }
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int u = 0; u < U; ++u) sum += exp2f(z[u] - ref);
    s = s * exp2f(m - ref) + sum;
    m = top;
    if (__any_sync(0xffffffffu, s != s)) return make_float2(m, NAN);
  }
  const float top = L::max_over_rows(m);
  return make_float2(top, L::over_rows(s * exp2f(m - (top == -INFINITY ? 0.f : top))));
}
// The same with values: P V's features lane, lane + 32, .. as well, against that maximum.  (Where it ends early m and s are of the keys
// until then.)
template <int D> struct Redone {
  float m, s, o[D / 32];
};
template <int D> __device__ __noinline__ Redone<D> redo_softmax(const Args& a, int64_t nk, int r, int at, float slope2, int j0, int j1) {
  using L = Lanes<__nv_bfloat16, D>;
  constexpr int U = L::kSteps;
  LaneSums<__nv_bfloat16, D> sums;
  const __nv_bfloat16 *k = (const __nv_bfloat16*)a.kc + nk * a.capacity * D, *v = (const __nv_bfloat16*)a.vc + nk * a.capacity * D;
  const uint4 q = sums.load((const __nv_bfloat16*)a.q + (nk * a.group * a.nodes + r) * D, 0);
  float m = -INFINITY, s = 0.f;
  for (int j = j0; j < j1; j += U * L::R) {
    uint4 x[U], y[U];
    float z[U], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = min(j + u * L::R + sums.own, j1 - 1);
      x[u] = sums.load(k, key);
      y[u] = sums.load(v, key);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j + u * L::R + sums.own;
      const float dot = sums.dot(q, x[u]);
      z[u] = key < j1 ? score<true>(dot, a.scale, a.cap, slope2, (float)(at - key)) : -INFINITY;
      top = fmaxf(top, z[u]);
    }
    const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m - ref);
    m = top;
    s *= f;
    sums.scale(f);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * L::R + sums.own < j1) {
        const float p = exp2f(z[u] - ref);
        s += p;
        sums.add(p, y[u]);
      }
    if (__any_sync(0xffffffffu, s != s) || sums.no_number()) break;
  }
  const float top = L::max_over_rows(m), f = exp2f(m - (top == -INFINITY ? 0.f : top));
  s = L::over_rows(s * f);
  sums.scale(f);
  sums.join(1.f);
  const int lane = threadIdx.x & 31;
  Redone<D> got{top, s, {}};
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int c = 0; c < L::E; ++c) {
      const float x = __shfl_sync(0xffffffffu, sums.x[c], (lane + 32 * e) / L::E);
      if (lane % L::E == c) got.o[e] = x;
    }
  return got;
}

// The accepted branch: what tree_accept writes.  path: (batch or 1, accepted) nodes.
struct Accept {
  const int* path;
  int64_t path_stride;
  int accepted;
  float* advanced;         // (batch, kv_heads, capacity), or null: no demand is kept
  void* kc;
  void* vc;
};

// The node of place x of the path, held inside the tree.
__device__ __forceinline__ int path_node(const Args& a, const Accept& c, int b, int x) {
  return min(max(c.path[b * c.path_stride + x], 0), a.nodes - 1);
}

}  // namespace tree
}  // namespace dil
