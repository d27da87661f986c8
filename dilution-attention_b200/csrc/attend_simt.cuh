// Softmax attention with caps, biases and masks (attend_common.cuh) on tiles of 64 queries by 64 keys with fp32 FMAs: fp32
// tensors, and bf16 heads that the tensor-core kernels do not take.  256 threads; thread (ty, tx) = (tid / 16, tid % 16)
// holds the scores of rows 4 ty .. 4 ty + 3 and columns tx, tx + 16, .. of a tile, and the accumulators of its rows and
// features tx, tx + 16, ..  Operand tiles lie in shared memory in fp32 with rows of D + 4 words, so that the 16 rows
// that a half warp reads at a time start in different banks.  Tiles without a visible pair are passed over.
#pragma once

#include "attend_common.cuh"

namespace dil {
namespace attend {

constexpr int kTile = 64;
constexpr int kSimtThreads = 256;

// Rows [r0, r0 + 64) of a (t, D) matrix into a tile, zeros behind the last.
template <typename T, int D>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int r0, int t) {
  constexpr int E = 16 / sizeof(T);
  for (int x = threadIdx.x; x < kTile * D / E; x += kSimtThreads) {
    const int row = x / (D / E), c = x % (D / E) * E;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r0 + row < t) w = *reinterpret_cast<const uint4*>(src + (int64_t)(r0 + row) * D + c);
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

template <int D> constexpr int simt_smem(int tiles) { return 4 * (tiles * kTile * (D + 4) + kTile * (kTile + 4)); }

// grid = batch * heads * ceil(t / 64), last query tiles (the longest) first.
template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) simt_forward_kernel(Args a) {
  extern __shared__ float sm[];
  float *sQ = sm, *sK = sQ + kTile * (D + 4), *sV = sK + kTile * (D + 4), *sP = sV + kTile * (D + 4);
  const int tiles = (a.t + kTile - 1) / kTile, heads = a.batch * a.heads;
  const int64_t n = blockIdx.x % heads;
  const int i0 = (tiles - 1 - (int)(blockIdx.x / heads)) * kTile;
  const int b = (int)(n / a.heads), h = (int)(n % a.heads);
  const int64_t nk = (int64_t)b * a.kv_heads + h / (a.heads / a.kv_heads);
  const Row r = make_row(a, b, h);
  const T* k = row_ptr<T>(a.k, nk, a.t, D);
  const T* v = row_ptr<T>(a.v, nk, a.t, D);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  load_tile<T, D>(sQ, row_ptr<T>(a.q, n, a.t, D), i0, a.t);
  float m[4], l[4], o[4][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[i][c] = 0.f;
  }
  const int end = key_end(r, min(i0 + kTile, a.t) - 1);
  for (int j0 = 0; j0 < end; j0 += kTile) {
    if (!tile_visible(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1)) continue;
    __syncthreads();
    load_tile<T, D>(sK, k, j0, a.t);
    load_tile<T, D>(sV, v, j0, a.t);
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
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = i0 + 4 * ty + i;
    const float sum = sum16(l[i]), inv = sum == 0.f ? 0.f : 1.f / sum;
    if (qi >= a.t) continue;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const float x = o[i][c] * inv;
      bad = bad || !isfinite(x);
      reinterpret_cast<T*>(a.out)[(n * a.t + qi) * D + tx + 16 * c] = from_f32<T>(x);
    }
    if (a.lse != nullptr && tx == 0) a.lse[n * a.t + qi] = sum == 0.f ? INFINITY : m[i] + log2f(sum);
  }
  if (__any_sync(0xffffffffu, bad))          // the 8 rows of this warp
    for (int x = 0; x < 8; ++x)
      if (i0 + 8 * (tid >> 5) + x < a.t) redo_forward_row<T, D>(a, b, h, i0 + 8 * (tid >> 5) + x);
}

// dq.  grid as above.
template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) simt_dq_kernel(Args a) {
  extern __shared__ float sm[];
  float *sQ = sm, *sG = sQ + kTile * (D + 4), *sX = sG + kTile * (D + 4), *sP = sX + kTile * (D + 4);
  const int tiles = (a.t + kTile - 1) / kTile, heads = a.batch * a.heads;
  const int64_t n = blockIdx.x % heads;
  const int i0 = (tiles - 1 - (int)(blockIdx.x / heads)) * kTile;
  const int b = (int)(n / a.heads), h = (int)(n % a.heads);
  const int64_t nk = (int64_t)b * a.kv_heads + h / (a.heads / a.kv_heads);
  const Row r = make_row(a, b, h);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  load_tile<T, D>(sQ, row_ptr<T>(a.q, n, a.t, D), i0, a.t);
  load_tile<T, D>(sG, row_ptr<T>(a.dout, n, a.t, D), i0, a.t);
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
  for (int j0 = 0; j0 < end; j0 += kTile) {
    if (!tile_visible(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1)) continue;
    float s[4][4], g[4][4];
    __syncthreads();
    load_tile<T, D>(sX, row_ptr<T>(a.v, nk, a.t, D), j0, a.t);
    __syncthreads();
    tile_scores<D>(sG, sX, ty, tx, g);
    __syncthreads();
    load_tile<T, D>(sX, row_ptr<T>(a.k, nk, a.t, D), j0, a.t);
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
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = i0 + 4 * ty + i;
    if (qi >= a.t) continue;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const float x = dq[i][c] * a.scale;
      bad = bad || !isfinite(x);
      reinterpret_cast<T*>(a.dq)[(n * a.t + qi) * D + tx + 16 * c] = from_f32<T>(x);
    }
  }
  if (__any_sync(0xffffffffu, bad))
    for (int x = 0; x < 8; ++x)
      if (i0 + 8 * (tid >> 5) + x < a.t) redo_dq_row<T, D>(a, b, h, i0 + 8 * (tid >> 5) + x);
}

// dk and dv of 64 keys of a key head, over all queries of the heads that share it.  Rows of a tile are keys here.
// grid = batch * kv_heads * ceil(t / 64), first key tiles (the longest) first.
template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) simt_dkv_kernel(Args a) {
  extern __shared__ float sm[];
  float *sK = sm, *sV = sK + kTile * (D + 4), *sX = sV + kTile * (D + 4), *sP = sX + kTile * (D + 4);
  const int heads = a.batch * a.kv_heads, group = a.heads / a.kv_heads;
  const int64_t nk = blockIdx.x % heads;
  const int j0 = (int)(blockIdx.x / heads) * kTile;
  const int b = (int)(nk / a.kv_heads), hk = (int)(nk % a.kv_heads);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  load_tile<T, D>(sK, row_ptr<T>(a.k, nk, a.t, D), j0, a.t);
  load_tile<T, D>(sV, row_ptr<T>(a.v, nk, a.t, D), j0, a.t);
  float dk[4][D / 16], dv[4][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < D / 16; ++c) dk[i][c] = dv[i][c] = 0.f;
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const Row r = make_row(a, b, h);
    const int64_t n = (int64_t)b * a.heads + h;
    for (int i0 = first_query(r, j0) / kTile * kTile; i0 < a.t; i0 += kTile) {
      if (!tile_visible(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1)) continue;
      float s[4][4], g[4][4];
      const bool full = tile_full(r, i0, i0 + kTile - 1, j0, j0 + kTile - 1);
      __syncthreads();
      load_tile<T, D>(sX, row_ptr<T>(a.q, n, a.t, D), i0, a.t);
      __syncthreads();
      tile_scores<D>(sK, sX, ty, tx, s);
      __syncthreads();
      load_tile<T, D>(sX, row_ptr<T>(a.dout, n, a.t, D), i0, a.t);
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
      load_tile<T, D>(sX, row_ptr<T>(a.q, n, a.t, D), i0, a.t);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sP[(4 * ty + i) * (kTile + 4) + tx + 16 * j] = s[i][j];
      __syncthreads();
      tile_accumulate<D>(sP, sX, ty, tx, dk);
    }
  }
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int kj = j0 + 4 * ty + i;
    if (kj >= a.t) continue;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const float x = dk[i][c] * a.scale, y = dv[i][c];
      bad = bad || !isfinite(x) || !isfinite(y);
      reinterpret_cast<T*>(a.dk)[(nk * a.t + kj) * D + tx + 16 * c] = from_f32<T>(x);
      reinterpret_cast<T*>(a.dv)[(nk * a.t + kj) * D + tx + 16 * c] = from_f32<T>(y);
    }
  }
  if (__any_sync(0xffffffffu, bad))
    for (int x = 0; x < 8; ++x)
      if (j0 + 8 * (tid >> 5) + x < a.t) redo_dkv_row<T, D>(a, b, hk, j0 + 8 * (tid >> 5) + x);
}

}  // namespace attend
}  // namespace dil
