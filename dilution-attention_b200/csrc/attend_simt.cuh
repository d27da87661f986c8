// Softmax attention with caps, biases and masks (attend_common.cuh) on tiles of 64 queries by 64 keys with fp32 FMAs: fp32
// tensors, and bf16 heads that the tensor-core kernels do not take.  256 threads; thread (ty, tx) = (tid / 16, tid % 16)
// holds the scores of rows 4 ty .. 4 ty + 3 and columns tx, tx + 16, .. of a tile, and the accumulators of its rows and
// features tx, tx + 16, ..  Operand tiles lie in shared memory in fp32 with rows of D + 4 words, so that the 16 rows
// that a half warp reads at a time start in different banks.  Tiles without a visible pair are passed over.
// Calls of few blocks share each block between the CTAs of a cluster: every `ranks`-th tile is a CTA's, and what they have
// accumulated is joined through distributed shared memory, in the ranks' order, each rank finishing a part of the rows.
// One sequence of 301 tokens, 4 heads of 64 (2 key heads), fp32, forward / dk, dv / dq: 38 / 95 / 38 us by one CTA a block,
// 23 / 26 / 19 us by clusters, whose length is then a tile's latency (loads, 64 x 64 x D FMAs twice, three barriers).
#pragma once

#include "attend_common.cuh"

namespace dil {
namespace attend {

constexpr int kTile = 64;
constexpr int kSimtThreads = 256;

// Rows [r0, r0 + 64) of a (t, D) matrix into a tile, zeros behind the last and in place of padding (docs, if not null, below 0).
template <typename T, int D>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int r0, int t, const int* docs) {
  constexpr int E = 16 / sizeof(T);
  for (int x = threadIdx.x; x < kTile * D / E; x += kSimtThreads) {
    const int row = x / (D / E), c = x % (D / E) * E;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r0 + row < t && (docs == nullptr || docs[r0 + row] >= 0)) w = *reinterpret_cast<const uint4*>(src + (int64_t)(r0 + row) * D + c);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < E; ++i) dst[row * (D + 4) + c + i] = to_f32(e[i]);
  }
}

// s[4][4] = A B^T for the thread's rows of A and columns (rows of B).
template <int D>
__device__ __forceinline__ void tile_scores(const float* a, const float* b, int ty, int tx, float s[4][4]) {
#pragma unroll
  for (int x = 0; x < 16; ++x) s[x >> 2][x & 3] = 0.f;
#pragma unroll 4
  for (int c = 0; c < D; c += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * (D + 4) + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * (D + 4) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
        s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
        s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
        s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
      }
  }
}

// acc[4][D / 16] += W X for rows 4 ty .. of W [64][68] and features tx + 16 c of X.
template <int D>
__device__ __forceinline__ void tile_accumulate(const float* w, const float* x, int ty, int tx, float acc[4][D / 16]) {
#pragma unroll 4
  for (int j = 0; j < kTile; ++j) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = w[(4 * ty + i) * (kTile + 4) + j];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const float v = x[j * (D + 4) + tx + 16 * c];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][c] = fmaf(p[i], v, acc[i][c]);
    }
  }
}

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

// Accumulators [4][D / 16] of a thread into a [64][D + 4] tile.
template <int D> __device__ __forceinline__ void put_tile(float* dst, int ty, int tx, const float acc[4][D / 16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < D / 16; ++c) dst[(4 * ty + i) * (D + 4) + tx + 16 * c] = acc[i][c];
}
// The rows' sums over the ranks of element x of their tiles.
__device__ __forceinline__ float over_ranks(const float* x, int ranks) {
  if (ranks == 1) return *x;
  float s = 0.f;
  for (int r = 0; r < ranks; ++r) s += ld_cluster(x, r);
  return s;
}
__device__ __forceinline__ void meet(int ranks) {
  if (ranks > 1) cluster_sync(); else __syncthreads();
}
// The rank's rows whose flag is set once more, by whole warps; a row's flag is its thread block's own.
template <Redo WHAT, typename T, int D>
__device__ __forceinline__ void redo_flagged(const Args& a, int b, int h, int r0, const int* flag, int first, int last) {
  __syncthreads();
  for (int row = first + (int)(threadIdx.x >> 5); row < last; row += kSimtThreads / 32)
    if (flag[row]) redo_rows<WHAT, T, D>(a, b, h, r0 + row, 1u);
}

template <int D> constexpr int simt_smem(int tiles) { return 4 * (tiles * kTile * (D + 4) + kTile * (kTile + 4)); }

// grid = ranks * batch * heads * ceil(t / 64), last query tiles (the longest) first.
template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) simt_forward_kernel(Args a, int ranks) {
  extern __shared__ float sm[];
  float *sQ = sm, *sK = sQ + kTile * (D + 4), *sV = sK + kTile * (D + 4), *sP = sV + kTile * (D + 4);
  const int tiles = (a.t + kTile - 1) / kTile, heads = a.batch * a.heads;
  const int rank = blockIdx.x % ranks, block = blockIdx.x / ranks;
  const int64_t n = block % heads;
  const int i0 = (tiles - 1 - block / heads) * kTile;
  const int b = (int)(n / a.heads), h = (int)(n % a.heads);
  const int64_t nk = (int64_t)b * a.kv_heads + h / (a.heads / a.kv_heads);
  const Row r = make_row(a, b, h);
  const T* k = row_ptr<T>(a.k, nk, a.t, D);
  const T* v = row_ptr<T>(a.v, nk, a.t, D);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  load_tile<T, D>(sQ, row_ptr<T>(a.q, n, a.t, D), i0, a.t, nullptr);
  float m[4], l[4], o[4][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[i][c] = 0.f;
  }
  const int end = key_end(r, min(i0 + kTile, a.t) - 1);
  int turn = 0;
  for (int j0 = 0; j0 < end; j0 += kTile) {
    if (!tile_visible(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1) || turn++ % ranks != rank) continue;
    __syncthreads();
    load_tile<T, D>(sK, k, j0, a.t, nullptr);
    load_tile<T, D>(sV, v, j0, a.t, r.docs);
    __syncthreads();
    float s[4][4];
    tile_scores<D>(sQ, sK, ty, tx, s);
    const bool full = tile_full(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int qi = i0 + 4 * ty + i;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int kj = j0 + tx + 16 * j;
        s[i][j] = full || sees(r, qi, kj) ? score<sizeof(T) == 4>(r, s[i][j], qi, kj).x : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      top = fmaxf(m[i], max16(top));
      const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m[i] - ref);
      m[i] = top;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - ref);
        sum += p;
        sP[(4 * ty + i) * (kTile + 4) + tx + 16 * j] = p;
      }
      l[i] = l[i] * f + sum;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) o[i][c] *= f;
    }
    __syncwarp();                    // a row's 16 threads are one half warp: P is handed over within it
    tile_accumulate<D>(sP, sV, ty, tx, o);
  }
  // [64] maxima, sums and flags over P, the accumulator over K
  __syncthreads();
  float *sM = sP, *sL = sP + kTile;
  int* sFlag = reinterpret_cast<int*>(sP + 2 * kTile);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float sum = sum16(l[i]);
    if (tx == 0) {
      sM[4 * ty + i] = m[i];
      sL[4 * ty + i] = sum;
      sFlag[4 * ty + i] = 0;
    }
  }
  put_tile<D>(sK, ty, tx, o);
  meet(ranks);
  const int part = kTile / ranks, first = rank * part, last = min(first + part, a.t - i0);
  for (int x = tid; x < (last - first) * D; x += kSimtThreads) {
    const int row = first + x / D, c = x % D;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
    for (int y = 0; y < ranks; ++y) top = fmaxf(top, ranks == 1 ? sM[row] : ld_cluster(sM + row, y));
    const float ref = top == -INFINITY ? 0.f : top;
    for (int y = 0; y < ranks; ++y) {
      const float f = exp2f((ranks == 1 ? sM[row] : ld_cluster(sM + row, y)) - ref);
      sum = fmaf(ranks == 1 ? sL[row] : ld_cluster(sL + row, y), f, sum);
      acc = fmaf(ranks == 1 ? sK[row * (D + 4) + c] : ld_cluster(sK + row * (D + 4) + c, y), f, acc);
    }
    const float out = sum == 0.f ? 0.f : acc / sum;
    if (!isfinite(out)) sFlag[row] = 1;
    reinterpret_cast<T*>(a.out)[(n * a.t + i0 + row) * D + c] = from_f32<T>(out);
    if (a.rest != nullptr) reinterpret_cast<T*>(a.rest)[(n * a.t + i0 + row) * D + c] = from_f32<T>(left_off<T>(out));
    if (a.lse != nullptr && c == 0) a.lse[n * a.t + i0 + row] = sum == 0.f ? INFINITY : top + log2f(sum);
  }
  redo_flagged<kRedoForward, T, D>(a, b, h, i0, sFlag, first, last);
  meet(ranks);                       // no CTA leaves while another may read its sums
}

// dq.  grid as above.
template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) simt_dq_kernel(Args a, int ranks) {
  extern __shared__ float sm[];
  float *sQ = sm, *sG = sQ + kTile * (D + 4), *sX = sG + kTile * (D + 4), *sP = sX + kTile * (D + 4);
  const int tiles = (a.t + kTile - 1) / kTile, heads = a.batch * a.heads;
  const int rank = blockIdx.x % ranks, block = blockIdx.x / ranks;
  const int64_t n = block % heads;
  const int i0 = (tiles - 1 - block / heads) * kTile;
  const int b = (int)(n / a.heads), h = (int)(n % a.heads);
  const int64_t nk = (int64_t)b * a.kv_heads + h / (a.heads / a.kv_heads);
  const Row r = make_row(a, b, h);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  load_tile<T, D>(sQ, row_ptr<T>(a.q, n, a.t, D), i0, a.t, nullptr);
  load_tile<T, D>(sG, row_ptr<T>(a.dout, n, a.t, D), i0, a.t, nullptr);
  float lse[4], delta[4], dq[4][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = i0 + 4 * ty + i;
    lse[i] = qi < a.t ? a.lse[n * a.t + qi] : INFINITY;
    delta[i] = qi < a.t ? a.delta[n * a.t + qi] : 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) dq[i][c] = 0.f;
  }
  const int end = key_end(r, min(i0 + kTile, a.t) - 1);
  int turn = 0;
  for (int j0 = 0; j0 < end; j0 += kTile) {
    if (!tile_visible(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1) || turn++ % ranks != rank) continue;
    float s[4][4], g[4][4];
    __syncthreads();
    load_tile<T, D>(sX, row_ptr<T>(a.v, nk, a.t, D), j0, a.t, r.docs);
    __syncthreads();
    tile_scores<D>(sG, sX, ty, tx, g);
    __syncthreads();
    load_tile<T, D>(sX, row_ptr<T>(a.k, nk, a.t, D), j0, a.t, r.docs);
    __syncthreads();
    tile_scores<D>(sQ, sX, ty, tx, s);
    const bool full = tile_full(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int qi = i0 + 4 * ty + i, kj = j0 + tx + 16 * j;
        float ds = 0.f;
        if (full || sees(r, qi, kj)) {
          const float2 z = score<sizeof(T) == 4>(r, s[i][j], qi, kj);
          ds = exp2f(z.x - lse[i]) * (g[i][j] - delta[i]) * z.y;
        }
        sP[(4 * ty + i) * (kTile + 4) + tx + 16 * j] = ds;
      }
    __syncwarp();
    tile_accumulate<D>(sP, sX, ty, tx, dq);
  }
  __syncthreads();
  int* sFlag = reinterpret_cast<int*>(sP);
  if (tid < kTile) sFlag[tid] = 0;
  put_tile<D>(sX, ty, tx, dq);
  meet(ranks);
  const int part = kTile / ranks, first = rank * part, last = min(first + part, a.t - i0);
  for (int x = tid; x < (last - first) * D; x += kSimtThreads) {
    const int row = first + x / D, c = x % D;
    const float y = over_ranks(sX + row * (D + 4) + c, ranks) * a.scale;
    if (!isfinite(y)) sFlag[row] = 1;
    reinterpret_cast<T*>(a.dq)[(n * a.t + i0 + row) * D + c] = from_f32<T>(y);
  }
  redo_flagged<kRedoDq, T, D>(a, b, h, i0, sFlag, first, last);
  meet(ranks);
}

// dk and dv of 64 keys of a key head, over all queries of the heads that share it.  Rows of a tile are keys here.
// grid = ranks * batch * kv_heads * ceil(t / 64), first key tiles (the longest) first.
template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) simt_dkv_kernel(Args a, int ranks) {
  extern __shared__ float sm[];
  float *sK = sm, *sV = sK + kTile * (D + 4), *sX = sV + kTile * (D + 4), *sP = sX + kTile * (D + 4);
  const int heads = a.batch * a.kv_heads, group = a.heads / a.kv_heads;
  const int rank = blockIdx.x % ranks, block = blockIdx.x / ranks;
  const int64_t nk = block % heads;
  const int j0 = block / heads * kTile;
  const int b = (int)(nk / a.kv_heads), hk = (int)(nk % a.kv_heads);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  load_tile<T, D>(sK, row_ptr<T>(a.k, nk, a.t, D), j0, a.t, nullptr);
  load_tile<T, D>(sV, row_ptr<T>(a.v, nk, a.t, D), j0, a.t, nullptr);
  float dk[4][D / 16], dv[4][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < D / 16; ++c) dk[i][c] = dv[i][c] = 0.f;
  int turn = 0;
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const Row r = make_row(a, b, h);
    const int64_t n = (int64_t)b * a.heads + h;
    for (int i0 = first_query(r, j0) / kTile * kTile; i0 < a.t; i0 += kTile) {
      if (!tile_visible(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1) || turn++ % ranks != rank) continue;
      float s[4][4], g[4][4];
      const bool full = tile_full(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1);
      __syncthreads();
      load_tile<T, D>(sX, row_ptr<T>(a.q, n, a.t, D), i0, a.t, r.docs);
      __syncthreads();
      tile_scores<D>(sK, sX, ty, tx, s);
      __syncthreads();
      load_tile<T, D>(sX, row_ptr<T>(a.dout, n, a.t, D), i0, a.t, r.docs);
      __syncthreads();
      tile_scores<D>(sV, sX, ty, tx, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {                  // the thread's queries
        const int qi = i0 + tx + 16 * j;
        const float lse = qi < a.t ? a.lse[n * a.t + qi] : INFINITY, delta = qi < a.t ? a.delta[n * a.t + qi] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kj = j0 + 4 * ty + i;
          float p = 0.f, ds = 0.f;
          if (full || sees(r, qi, kj)) {
            const float2 z = score<sizeof(T) == 4>(r, s[i][j], qi, kj);
            p = exp2f(z.x - lse);
            ds = p * (g[i][j] - delta) * z.y;
          }
          sP[(4 * ty + i) * (kTile + 4) + tx + 16 * j] = p;
          s[i][j] = ds;
        }
      }
      __syncwarp();
      tile_accumulate<D>(sP, sX, ty, tx, dv);
      __syncthreads();
      load_tile<T, D>(sX, row_ptr<T>(a.q, n, a.t, D), i0, a.t, r.docs);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sP[(4 * ty + i) * (kTile + 4) + tx + 16 * j] = s[i][j];
      __syncthreads();
      tile_accumulate<D>(sP, sX, ty, tx, dk);
    }
  }
  __syncthreads();
  int* sFlag = reinterpret_cast<int*>(sP);
  if (tid < kTile) sFlag[tid] = 0;
  put_tile<D>(sK, ty, tx, dk);
  put_tile<D>(sV, ty, tx, dv);
  meet(ranks);
  const int part = kTile / ranks, first = rank * part, last = min(first + part, a.t - j0);
  for (int x = tid; x < (last - first) * D; x += kSimtThreads) {
    const int row = first + x / D, c = x % D;
    const float y = over_ranks(sK + row * (D + 4) + c, ranks) * a.scale, z = over_ranks(sV + row * (D + 4) + c, ranks);
    if (!isfinite(y) || !isfinite(z)) sFlag[row] = 1;
    reinterpret_cast<T*>(a.dk)[(nk * a.t + j0 + row) * D + c] = from_f32<T>(y);
    reinterpret_cast<T*>(a.dv)[(nk * a.t + j0 + row) * D + c] = from_f32<T>(z);
  }
  redo_flagged<kRedoDkv, T, D>(a, b, hk, j0, sFlag, first, last);
  meet(ranks);
}

}  // namespace attend
}  // namespace dil
