// Tree steps with fp32 FMAs, for fp32 caches and the head sizes that the tensor-core kernels do not take.
//
// 256 threads walk a chunk of a key head's keys in tiles of 64; 16 RI of its rows are held at a time: thread
// (ty, tx) = (tid / 16, tid % 16) has rows ty + 16 i and keys tx + 16 j of a tile.  A step's chunks are joined by
// join_kernel.  What bounds them is the cache's bytes: at RI = 1 a tile of 64 keys takes 16 x 64 x D x 2 FMAs, which the
// SM does in less time than its share of the memory system needs for the tile; from RI = 2 on the FMAs are the bound.
// 16 heads of 32, 40 nodes over 4099 keys, fp32: statistics 21, shares 43, five accepted nodes' bids 10 us; the cache's 17 MB take 2.6.
#pragma once

#include "tree_common.cuh"

namespace dil {
namespace tree {

constexpr int kKeys = 64;
constexpr int kThreads = 256;

template <typename T, int D>
__device__ __forceinline__ void load_rows(float* dst, const T* const* src, int rows) {
  constexpr int E = 16 / sizeof(T);
  for (int x = threadIdx.x; x < rows * D / E; x += kThreads) {
    const int row = x / (D / E), c = x % (D / E) * E;
    const T* p = src[row];
    uint4 w = make_uint4(0, 0, 0, 0);
    if (p != nullptr) w = *reinterpret_cast<const uint4*>(p + c);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < E; ++i) dst[row * (D + 4) + c + i] = to_f32(e[i]);
  }
}

template <int D, int RI> struct Smem {
  float q[16 * RI * (D + 4)];
  float x[kKeys * (D + 4)];
  float p[16 * RI * (kKeys + 4)];
  float had[16 * RI * (kKeys + 4)];
  Lineage tree;
  const void* qrow[16 * RI];
  const void* krow[kKeys];
  int node[kKeys];            // the node of a key, -1 for a cached one, -2 for none
};

template <typename T, int D, int RI> struct Walker {
  using S = Smem<D, RI>;
  const Args& a;
  S& s;
  int b, hk, len, rows, ty, tx;
  int64_t nk;
  __device__ Walker(const Args& args, S& smem, int64_t row) : a(args), s(smem), nk(row) {
    b = (int)(row / a.kv_heads);
    hk = (int)(row % a.kv_heads);
    len = cache_len(a.pos_dev, a.len, a.capacity);
    rows = a.group * a.nodes;
    ty = threadIdx.x >> 4;
    tx = threadIdx.x & 15;
    make_lineage(&s.tree, a.parents + b * a.parent_stride, a.nodes);
  }
  // Rows [r0, r0 + 16 RI) of the queries; `pick` gives the row of a place, or -1.
  template <typename Pick> __device__ void queries(Pick pick) {
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * RI; x += kThreads) {
      const int r = pick(x);
      s.qrow[x] = r >= 0 ? (const T*)a.q + (nk * rows + r) * D : nullptr;
    }
    __syncthreads();
    load_rows<T, D>(s.q, reinterpret_cast<const T* const*>(s.qrow), 16 * RI);
  }
  // Where keys [j0, j1) of a tile come from, K or V; `node` gives the node of key len + x.
  template <typename Node> __device__ void keys(bool values, int j0, int j1, Node node) {
    __syncthreads();
    for (int x = threadIdx.x; x < kKeys; x += kThreads) {
      const int j = j0 + x, at = j >= j1 ? -2 : j < len ? -1 : node(j - len);
      const T* cache = (const T*)(values ? a.vc : a.kc);
      const T* drafted = (const T*)(values ? a.vn : a.kn);
      s.krow[x] = at == -2 ? nullptr : at == -1 ? cache + (nk * a.capacity + j) * D : drafted + (nk * a.nodes + at) * D;
      s.node[x] = at;
    }
    __syncthreads();
    load_rows<T, D>(s.x, reinterpret_cast<const T* const*>(s.krow), kKeys);
    __syncthreads();
  }
  __device__ void products(float z[RI][4]) {
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) z[i][j] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
      float4 y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(s.x + (tx + 16 * j) * (D + 4) + c);
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(s.q + (ty + 16 * i) * (D + 4) + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          z[i][j] = fmaf(x.x, y[j].x, z[i][j]);
          z[i][j] = fmaf(x.y, y[j].y, z[i][j]);
          z[i][j] = fmaf(x.z, y[j].z, z[i][j]);
          z[i][j] = fmaf(x.w, y[j].w, z[i][j]);
        }
      }
    }
  }
  // The scores of row r (node % nodes) against the tile's keys from j0 on; -inf where it does not see the key.
  __device__ void scores(int r, int j0, float z[4]) {
    if (j0 + kKeys <= len && a.cap == 0.f && a.slopes == nullptr) {       // (rows behind the last go nowhere)
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] *= a.scale * kLog2e;
      return;
    }
    const int x = r >= 0 ? r % a.nodes : 0, h = hk * a.group + (r >= 0 ? r / a.nodes : 0);
    const float slope2 = a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
    const int at = s.tree.depth[x];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int y = s.node[tx + 16 * j];
      const bool ok = r >= 0 && (y == -1 || (y >= 0 && (s.tree.line[x] >> y & 1)));
      const float far = (float)(y >= 0 ? at - s.tree.depth[y] : len + at - (j0 + tx + 16 * j));
      z[j] = ok ? score<sizeof(T) == 4>(z[j], a.scale, a.cap, slope2, far) : -INFINITY;
    }
  }
  // acc += P X; a share of zero passes over its value, which a masked node need not have finite (tiles with nodes only)
  __device__ void accumulate(bool nodes, float acc[RI][D / 16]) {
    auto turn = [&](auto careful) {
#pragma unroll 4
      for (int j = 0; j < kKeys; ++j) {
        float p[RI];
#pragma unroll
        for (int i = 0; i < RI; ++i) p[i] = s.p[(ty + 16 * i) * (kKeys + 4) + j];
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const float v = s.x[j * (D + 4) + tx + 16 * c];
#pragma unroll
          for (int i = 0; i < RI; ++i) acc[i][c] = fmaf(p[i], decltype(careful)::value && p[i] == 0.f ? 0.f : v, acc[i][c]);
        }
      }
    };
    if (nodes) turn(std::true_type{}); else turn(std::false_type{});
  }
};

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Online softmax over a chunk: (maximum, sum) of every row and, if OUT, its part of P V.
// grid = (chunks, ceil(rows / 16 RI), batch * kv_heads)
template <typename T, int D, int RI, bool OUT>
__global__ void __launch_bounds__(kThreads) simt_softmax_kernel(Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Walker<T, D, RI> w(a, *reinterpret_cast<Smem<D, RI>*>(raw), blockIdx.z);
  const int2 range = chunk_keys(w.len + a.nodes, a.chunks, blockIdx.x, kKeys);
  const int r0 = blockIdx.y * 16 * RI;
  auto row = [&](int x) { return r0 + x < w.rows ? r0 + x : -1; };
  auto node = [](int x) { return x; };
  w.queries(row);
  float m[RI], l[RI], o[RI][D / 16];
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[i][c] = 0.f;
  }
  for (int j0 = range.x; j0 < range.y; j0 += kKeys) {
    w.keys(false, j0, range.y, node);
    float z[RI][4];
    w.products(z);
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      w.scores(row(w.ty + 16 * i), j0, z[i]);
      const float top = fmaxf(m[i], max16(fmaxf(fmaxf(z[i][0], z[i][1]), fmaxf(z[i][2], z[i][3]))));
      const float ref = top == -INFINITY ? 0.f : top, f = fast_exp2(m[i] - ref);
      m[i] = top;
      l[i] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = fast_exp2(z[i][j] - ref);
        l[i] += p;
        if (OUT) w.s.p[(w.ty + 16 * i) * (kKeys + 4) + w.tx + 16 * j] = p;
      }
      if (OUT)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[i][c] *= f;
    }
    if (OUT) {
      w.keys(true, j0, range.y, node);
      w.accumulate(j0 + kKeys > w.len, o);
    }
  }
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    const int r = row(w.ty + 16 * i);
    const float sum = sum16(l[i]);
    if (r < 0) continue;
    const int64_t at = (w.nk * a.chunks + blockIdx.x) * w.rows + r;
    if (w.tx == 0) a.part[at] = make_float2(m[i], sum);
    if (OUT)
#pragma unroll
      for (int c = 0; c < D / 16; ++c) a.pout[at * D + w.tx + 16 * c] = o[i][c];
  }
}

// lse of every row from its chunks' statistics.  One warp per row.
__global__ void __launch_bounds__(256) join_stats_kernel(Args a) {
  const int rows = a.group * a.nodes, lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= (int64_t)a.batch * a.kv_heads * rows) return;
  const int64_t nk = at / rows;
  const float2* part = a.part + nk * a.chunks * rows + at % rows;
  float m = -INFINITY, s = 0.f;
  for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, part[(int64_t)c * rows].x);
  m = warp_max(m);
  for (int c = lane; c < a.chunks; c += 32) {
    const float2 x = part[(int64_t)c * rows];
    // (a part without a score of its own has a sum of 0; NaN is handed on)
    s += x.y == 0.f ? 0.f : x.y * exp2f(x.x - (m == -INFINITY ? 0.f : m));
  }
  s = warp_sum(s);
  if (lane == 0) a.lse[at] = (m == -INFINITY ? 0.f : m) + log2f(s);
}

// Output of every row from its chunks.  DILUTE: sum / (sum of shares + eps); otherwise the parts, each against its own
// maximum, and lse.  One block of D threads per row.
template <typename T, bool DILUTE>
__global__ void join_kernel(Args a, int d) {
  const int rows = a.group * a.nodes, c = threadIdx.x;
  const int64_t at = blockIdx.x, nk = at / rows;
  const int64_t first = nk * a.chunks * rows + at % rows;
  float m = -INFINITY, s = 0.f, o = 0.f;
  if (!DILUTE)
    for (int x = 0; x < a.chunks; ++x) m = fmaxf(m, a.part[first + (int64_t)x * rows].x);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int x = 0; x < a.chunks; ++x) {
    const int64_t y = first + (int64_t)x * rows;
    const float sum = DILUTE ? a.psum[y] : a.part[y].y;
    const float f = DILUTE ? 1.f : exp2f(a.part[y].x - ref);
    if (!DILUTE && sum == 0.f) continue;
    s = fmaf(f, sum, s);
    o = fmaf(f, a.pout[y * d + c], o);
  }
  reinterpret_cast<T*>(a.out)[at * d + c] = from_f32<T>(DILUTE ? o / (s + a.eps) : o / s);
  if (!DILUTE && c == 0) a.lse[at] = ref + log2f(s);
}

// Shares of a dilution layer's nodes and their part of share V.  Each key's demand is walked through the tree by one
// thread, in the nodes' order: a node's demand is its parent's demand and bid.
// grid = (chunks, 1, batch * heads); 16 RI >= nodes
template <typename T, int D, int RI>
__global__ void __launch_bounds__(kThreads) simt_dilute_kernel(Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Walker<T, D, RI> w(a, *reinterpret_cast<Smem<D, RI>*>(raw), blockIdx.z);
  const int2 range = chunk_keys(w.len + a.nodes, a.chunks, blockIdx.x, kKeys);
  auto row = [&](int x) { return x < a.nodes ? x : -1; };
  auto node = [](int x) { return x; };
  w.queries(row);
  float lse[RI], sum[RI], o[RI][D / 16];
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    lse[i] = row(w.ty + 16 * i) >= 0 ? a.lse[w.nk * a.nodes + w.ty + 16 * i] : 0.f;
    sum[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[i][c] = 0.f;
  }
  for (int j0 = range.x; j0 < range.y; j0 += kKeys) {
    w.keys(false, j0, range.y, node);
    float z[RI][4];
    w.products(z);
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      w.scores(row(w.ty + 16 * i), j0, z[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) w.s.p[(w.ty + 16 * i) * (kKeys + 4) + w.tx + 16 * j] = fast_exp2(z[i][j] - lse[i]);
    }
    __syncthreads();
    // the demand behind every node, by one thread per key; then the shares, by all
    if (threadIdx.x < kKeys) {
      const int key = threadIdx.x, j = j0 + key;
      const float base = j < w.len ? a.committed[w.nk * a.capacity + j] : 0.f;
      float left = base;
#pragma unroll 4
      for (int x = 0; x < a.nodes; ++x) {
        const int up = w.s.tree.parent[x];
        if (up != x - 1 || up < 0) left = up >= 0 ? w.s.had[up * (kKeys + 4) + key] : base;
        left += w.s.p[x * (kKeys + 4) + key];
        w.s.had[x * (kKeys + 4) + key] = left;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = (w.ty + 16 * i) * (kKeys + 4) + w.tx + 16 * j;
        const float p = w.s.p[at];
        // (a node that does not see the key has no share of it, whatever the demand is)
        if (row(w.ty + 16 * i) >= 0) w.s.p[at] = p == 0.f ? 0.f : p / (w.s.had[at] + a.eps);
      }
    w.keys(true, j0, range.y, node);
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i] += w.s.p[(w.ty + 16 * i) * (kKeys + 4) + w.tx + 16 * j];
    w.accumulate(j0 + kKeys > w.len, o);
  }
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    const int r = row(w.ty + 16 * i);
    const float total = sum16(sum[i]);
    if (r < 0) continue;
    const int64_t at = (w.nk * a.chunks + blockIdx.x) * a.nodes + r;
    if (w.tx == 0) a.psum[at] = total;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) a.pout[at * D + w.tx + 16 * c] = o[i][c];
  }
}

// advanced_j = committed_j + the bids of the accepted nodes (of all heads that share the key head), for cached keys; the
// bids of one another for the accepted nodes' own keys.  grid = (blocks of tiles, 1, batch * kv_heads)
template <typename T, int D, int RI>
__global__ void __launch_bounds__(kThreads) simt_advance_kernel(Args a, Accept c) {
  extern __shared__ __align__(16) uint8_t raw[];
  Walker<T, D, RI> w(a, *reinterpret_cast<Smem<D, RI>*>(raw), blockIdx.z);
  const int keys = (int)min((int64_t)w.len + c.accepted, a.capacity), rows = a.group * c.accepted;
  auto node = [&](int x) { return path_node(a, c, w.b, x); };
  for (int j0 = blockIdx.x * kKeys; j0 < keys; j0 += gridDim.x * kKeys) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    w.keys(false, j0, keys, node);
    for (int r0 = 0; r0 < rows; r0 += 16 * RI) {
      auto row = [&](int x) { return r0 + x < rows ? (r0 + x) / c.accepted * a.nodes + node((r0 + x) % c.accepted) : -1; };
      w.queries(row);
      __syncthreads();
      float z[RI][4];
      w.products(z);
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        const int r = row(w.ty + 16 * i);
        w.scores(r, j0, z[i]);
        const float lse = r >= 0 ? a.lse[w.nk * w.rows + r] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += r >= 0 ? fast_exp2(z[i][j] - lse) : 0.f;
      }
    }
    // the 16 rows of threads, one after the other: the order is fixed
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) w.s.p[w.ty * (kKeys + 4) + w.tx + 16 * j] = sum[j];
    __syncthreads();
    if (threadIdx.x < kKeys && j0 + (int)threadIdx.x < keys) {
      const int64_t at = w.nk * a.capacity + j0 + threadIdx.x;
      float total = j0 + (int)threadIdx.x < w.len ? a.committed[at] : 0.f;
      for (int y = 0; y < 16; ++y) total += w.s.p[y * (kKeys + 4) + threadIdx.x];
      c.advanced[at] = total;
    }
  }
}

// The accepted nodes' keys and values behind the cache's last.  16 bytes a thread.
__global__ void __launch_bounds__(256) append_kernel(Args a, Accept c, int row_bytes) {
  const int per = row_bytes / 16, len = cache_len(a.pos_dev, a.len, a.capacity);
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, nk = at / per / c.accepted;
  const int x = (int)(at / per % c.accepted), u = (int)(at % per);
  if (nk >= (int64_t)a.batch * a.kv_heads || (int64_t)len + x >= a.capacity) return;
  const int node = path_node(a, c, (int)(nk / a.kv_heads), x);
  const int64_t src = (nk * a.nodes + node) * per + u, dst = (nk * a.capacity + len + x) * per + u;
  reinterpret_cast<uint4*>(c.kc)[dst] = reinterpret_cast<const uint4*>(a.kn)[src];
  reinterpret_cast<uint4*>(c.vc)[dst] = reinterpret_cast<const uint4*>(a.vn)[src];
}

}  // namespace tree
}  // namespace dil
