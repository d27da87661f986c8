// Drafted tokens over a cache: what the kernels of tree steps share.
//
// A tree of N <= 64 drafted nodes continues a cache of `len` keys.  Node x sees the cached keys, its ancestors and itself;
// it stands at position len + depth(x).  A key head's rows are the nodes of the `group` query heads that share it:
// row r is node r % N of head r / N.  Keys are numbered [0, len) in the cache and len + x for node x.
#pragma once

#include "common.cuh"

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
