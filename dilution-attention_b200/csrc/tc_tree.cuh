// Tree steps over a bf16 cache with heads of 64 and 128, on the tensor cores.  All nodes see all cached keys, so the kernels
// that stream the cache know no mask but its end; the nodes' own keys (64 at most) are joined in afterwards with fp32 FMAs.
//
//   scan_kernel : scores S = Q K^T, lane = row of the key head; online softmax, and P V if asked for.  Rows are few, lanes are
//                 128: up to 32 (64) rows are laid out four times (twice), each time against another quarter (half) of a tile's
//                 keys.  That is a product with a block-diagonal Q: the quarters' operands are one buffer with zeros around the
//                 rows, read from another offset, and each warp's P~ goes to columns of its own that are zero in other
//                 lanes.  The tensor pipe has the time (the cache's bytes are the bound), the special-function unit has not.
//   sweep_kernel: S^T = K Q^T, lane = key, for what belongs to keys: a thread walks the tree in the nodes' order with its
//                 key's demand (a node's demand is its parent's demand and bid; a parent further back is found in the TMEM
//                 column that its score came from), and out^T += V^T share; or it adds the accepted nodes' bids.
// What bounds them: the cache's bytes.  256 heads of 64, 24 nodes over 16384 keys: statistics 96 us (0.54 GB, 0.85 of the copy
// rate), shares and outputs 169 us (1.09 GB, 0.98), five accepted nodes' bids 86 us (0.55 GB, 0.98).  64 key heads whose 128 rows
// fill the lanes: 70 us for 0.27 GB, of which the exponentials need 30.
// A chunk of a key head's keys per CTA; one warp issues copies, one MMAs, two warpgroups take tiles in turn.
#pragma once

#include "tc_score.cuh"
#include "tree_common.cuh"

namespace dil {
namespace tc {

__device__ int g_tree_status = 0;          // first bounded wait that ran out (0 = none)

// 16 bytes c of row `row` of a [rows][64] bf16 tile under the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int c) { return (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)); }

__device__ __forceinline__ void tmem_st1(uint32_t taddr, float v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}

// A cache's tile whose last rows lie behind its end (a length that only the device knows: the copy could not leave them out).
__device__ __forceinline__ void zero_rows(uint8_t* tile, int rows, int from, int subs) {
  for (int s = 0; s < subs; ++s)
    for (int x = from * 8 + (int)(threadIdx.x & 31); x < rows * 8; x += 32)
      reinterpret_cast<uint4*>(tile + s * rows * 128)[x] = make_uint4(0, 0, 0, 0);
}

// Barriers of a CTA that streams a cache, keys through RK stages and values through RV, and scores it into NB buffers.  Keys
// are let go once they are scored, values by the product, which comes up to NB - 1 tiles later.  A buffer's scores are there
// (sdone) and have been used (ready); the last product of a warpgroup's values is through (used), and all are (alldone).
template <int RK, int RV, int NB> struct StreamBars {
  static_assert(NB <= RV + 1, "the copies of a tile's values never wait for a later tile's scores");
  uint32_t kfull, kfree, vfull, vfree, sdone, used, alldone, ready;
  Ctl* ctl;
  static constexpr int kBytes = 8 * (2 * RK + 2 * RV + 2 * NB + 3) + 16;
  __device__ __forceinline__ StreamBars(uint64_t* b) {
    kfull = smem_u32(b);
    kfree = kfull + 8 * RK;
    vfull = kfree + 8 * RK;
    vfree = vfull + 8 * RV;
    sdone = vfree + 8 * RV;
    used = sdone + 8 * NB;
    alldone = used + 16;
    ready = alldone + 8;
    ctl = reinterpret_cast<Ctl*>(b + 2 * RK + 2 * RV + 2 * NB + 3);
  }
  __device__ __forceinline__ void init() const {
    ctl->abort = 0;
    for (int x = 0; x < 2 * RK + 2 * RV + NB + 3; ++x) mbar_init(kfull + 8 * x, 1);
    for (int x = 0; x < NB; ++x) mbar_init(ready + 8 * x, 4);
    fence_barrier_init();
  }
};

// The warp that copies ne tiles of KT keys and (if V) their values: from, from + step, ..  Scans go from the last tile down: a
// distance bias has the largest scores there, and later tiles do not move a row's reference.
template <int D, int KT, int RK, int RV, int NB, bool V>
__device__ __forceinline__ void stream_tiles(const StreamBars<RK, RV, NB>& bars, const CUtensorMap* map_k, const CUtensorMap* map_v,
                                             uint32_t ring_k, uint32_t ring_v, int from, int step, int ne, int nk, uint32_t lead) {
  constexpr uint32_t kOne = KT * D * 2;
  auto copy = [&](const CUtensorMap* map, uint32_t dst, int e, uint32_t bar) {
    if (lead) {
      mbar_expect_tx(bar, kOne);
#pragma unroll
      for (int x = 0; x < KT / 64; ++x) tma_load_rows<kForm<D>>(dst + 8192 * x, map, (from + step * e) * KT + 64 * x, nk, bar, KT * 128);
    }
    __syncwarp();
  };
  for (int e = 0; e < ne; ++e) {
    const int k = e % RK, v = e % RV;
    if (e >= RK) mbar_wait_warp(bars.kfree + 8 * k, (e / RK - 1) & 1, bars.ctl, &g_tree_status, kErrWaitMma);
    copy(map_k, ring_k + kOne * k, e, bars.kfull + 8 * k);
    if (V) {
      if (e >= RV) mbar_wait_warp(bars.vfree + 8 * v, (e / RV - 1) & 1, bars.ctl, &g_tree_status, kErrWaitMma);
      copy(map_v, ring_v + kOne * v, e, bars.vfull + 8 * v);
    }
  }
}

// ---- scan ----------------------------------------------------------------------------------------------
// Registers, TMEM and shared memory of two CTAs on an SM: the start and the end of one overlap the other's tiles.
constexpr int ctas_per_sm(int bytes, int tmem) { return 2 * (bytes + 2304) <= 233472 && 2 * tmem <= 512 ? 2 : 1; }

template <int D, int G, bool OUT> struct Scan {
  // 64 columns a product, or 32 where P~ of several quarters is kept as well.  Statistics alone, 256 heads of 64, 24 nodes over 16384
  // keys: 32 columns 105 us, 64 columns 96 us: a product of few columns takes the tensor pipe nearly as long.
  static constexpr int kRows = 128 / G, kCols = G == 1 || !OUT ? 64 : 32, kKeys = kCols * G;
  static constexpr int kWg = OUT && D == 64 ? 1 : 2;                       // warpgroups, which take tiles in turn
  static constexpr int kThreads = 128 * kWg + 64;
  static constexpr uint32_t kOne = kKeys * D * 2;
  static constexpr int kSpace = D == 64 ? 65536 : 131072, kStages = (int)(kSpace / kOne) < 8 ? (int)(kSpace / kOne) : 8;
  static constexpr int kK = OUT ? kStages / 2 : kStages, kV = OUT ? kStages / 2 : 4;
  static constexpr int kBufRows = (G - 1) * kRows + 128;                   // zeros, the rows, zeros
  static constexpr uint32_t kBufSub = kBufRows * 128;
  static constexpr int kBuf = (int)kBufSub * (D / 64), kRingBytes = (int)kOne * kStages;
  static constexpr int kBytes = kBuf + kRingBytes + 2048 + 512 + 1024;
  // score buffers (tiles are scored ahead of the arithmetic), then P~ and the accumulator of each warpgroup
  static constexpr int kWgCols = OUT ? 64 + D : 0, kBuffers = OUT ? 2 : 4;
  static constexpr int kCols32 = kBuffers * kCols + kWg * kWgCols, kTmem = kCols32 <= 256 ? 256 : 512;
  static constexpr int kPerSm = ctas_per_sm(kBytes, kTmem);
  static_assert(kCols32 <= 512 && StreamBars<kK, kV, kBuffers>::kBytes <= 512, "score buffers");
  static_assert(!OUT || kWg * 128 * D * 4 <= kRingBytes, "the merge area fits the ring");
  static_assert(kK >= 2 && kBytes <= 231000, "shared memory");
};

// One warpgroup's step: kCols scores of a lane at tS, its P~ (OUT) to tP, in bf16, the values' type: each off by up to 2^-8 of itself,
// which out, divided by the sum of the others, carries (0.0023 by norm, where 0.0017 is the rounding of out alone).
template <int D, int N, bool OUT>
__device__ __forceinline__ void scan_step(uint32_t tS, uint32_t tP, uint32_t tO, float lin, float pre, bool cap, float slope2, float far, int valid,
                                          float& ref, float& s) {
  float v[N];
  uint32_t pw[N / 2];
  float ps;
  auto fetch = [&]() {
    tmem_ld32(tS, v);
    if (N == 64) tmem_ld32(tS + 32, v + (N - 32));
    tmem_ld_wait(v);
    if (N == 64) tmem_ld_wait(v + (N - 32));
    if (cap) cap_scores<N>(v, pre, lin > kWideCap * kLog2e);
    if (valid < N) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = e < valid ? v[e] : -INFINITY;
    }
  };
  // z = mul v + add + step e (the distance shrinks with the key's position)
  auto exponentials = [&](float mul, float add, float step) {
    const float2 mm = make_float2(mul, mul), four = make_float2(4.f * step, 4.f * step);
    float2 o0 = make_float2(add, add + step), o1 = make_float2(add + 2.f * step, add + 3.f * step);
    float2 a0 = make_float2(0.f, 0.f), a1 = a0;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float2 z0 = fma2(make_float2(v[e], v[e + 1]), mm, o0), z1 = fma2(make_float2(v[e + 2], v[e + 3]), mm, o1);
      o0 = add2(o0, four);
      o1 = add2(o1, four);
      const float2 p0 = make_float2(fast_exp2(z0.x), fast_exp2(z0.y)), p1 = make_float2(fast_exp2(z1.x), fast_exp2(z1.y));
      a0 = add2(a0, p0);
      a1 = add2(a1, p1);
      if (OUT) {
        pw[e >> 1] = pack_pair(p0.x, p0.y);
        pw[(e >> 1) + 1] = pack_pair(p1.x, p1.y);
      }
    }
    const float2 a = add2(a0, a1);
    ps = a.x + a.y;
  };
  const float add = -slope2 * far;
  fetch();
  bool slow = __any_sync(0xffffffffu, ref == -INFINITY && valid > 0);
  if (!slow) {
    exponentials(lin, ref == -INFINITY ? 0.f : add - ref, slope2);
    slow = __any_sync(0xffffffffu, !(ps < 1099511627776.f));       // 2^40
    if (slow) fetch();               // rare: the scores are still in TMEM
  }
  if (slow) {
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      v[e] = fmaf(v[e], lin, fmaf(slope2, (float)e, add));
      top = fmaxf(top, v[e]);
    }
    const float now = fmaxf(ref, top);
    if (__any_sync(0xffffffffu, now != ref)) {
      const bool fresh = __all_sync(0xffffffffu, ref == -INFINITY);
      const float f = fast_exp2(ref - (now == -INFINITY ? 0.f : now));
      if (OUT && !fresh) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float o[16];
          tmem_ld16(tO + 16 * c, o);
          tmem_ld_wait16(o);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * f);
          tmem_st16(tO + 16 * c, w);
        }
      }
      s *= f;
      ref = now;
    }
    exponentials(1.f, ref == -INFINITY ? 0.f : -ref, 0.f);
  }
  s += ps;
  if (OUT) {
    tmem_st16(tP, pw);
    if (N == 64) tmem_st16(tP + 16, pw + (N / 2 - 16));
    tmem_st_wait();
  }
}

// grid = (chunks, ceil(rows / 128) or 1, batch * kv_heads)
template <int D, int G, bool OUT>
__global__ void __launch_bounds__(Scan<D, G, OUT>::kThreads, Scan<D, G, OUT>::kPerSm) scan_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                      const __grid_constant__ tree::Args a) {
  using F = Scan<D, G, OUT>;
  constexpr int RK = F::kK, RV = F::kV, NB = F::kBuffers, NW = F::kWg, KT = F::kKeys, NC = F::kCols, SUB = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  const uint32_t sQ = smem_u32(smem), ring_k = sQ + F::kBuf, ring_v = ring_k + F::kOne * RK;
  float2* sStat = reinterpret_cast<float2*>(smem + F::kBuf + F::kRingBytes);              // [2][128]
  const StreamBars<RK, RV, NB> bars(reinterpret_cast<uint64_t*>(smem + F::kBuf + F::kRingBytes + 2048));
  Ctl* ctl = bars.ctl;
  __shared__ tree::Lineage lineage;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = tid >> 7, row = tid & 127;
  const int warp_u = uniform_warp();
  const uint32_t lead = elect_one();
  const int nk = blockIdx.z, b = nk / a.kv_heads, hk = nk % a.kv_heads, rows = a.group * a.nodes, r0 = blockIdx.y * 128;
  const int len = (int)uniform(tree::cache_len(a.pos_dev, a.len, a.capacity));
  const int2 keys = tree::chunk_keys(len, a.chunks, blockIdx.x, KT);
  const int ne = (keys.y - keys.x + KT - 1) / KT, last = keys.x / KT + ne - 1;

  let_next_in();
  if (tid == 0) bars.init();
  // the rows between zeros
  for (int x = tid; x < F::kBufRows * 8 * SUB; x += F::kThreads) {
    const int sub = x / (F::kBufRows * 8), br = x / 8 % F::kBufRows, c = x % 8, r = r0 + br - (G - 1) * F::kRows;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r >= r0 && r < min(rows, r0 + F::kRows))
      w = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + ((int64_t)nk * rows + r) * D + 64 * sub + 8 * c);
    *reinterpret_cast<uint4*>(smem + sub * F::kBufSub + swizzled(br, c)) = w;
  }
  fence_async_smem();
  if (a.slopes != nullptr) tree::make_lineage(&lineage, a.parents + b * a.parent_stride, a.nodes);
  __syncwarp();
  if (warp == 0) tmem_alloc(smem_u32(&ctl->tmem), F::kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl->tmem);

  if (warp_u == 4 * NW) {
    // ------------------------------------------------------------ the warp that issues MMAs
    constexpr uint32_t id_s = instr_desc(128, NC, 0, 0), id_p = instr_desc(128, D, 0, 1);
    const Desc dQ = make_desc(sQ, 16, 1024), dK = make_desc(ring_k, 16, 1024), dV = make_desc(ring_v, KT * 128, 1024);
    // what the compute warps clear (their P~ columns and accumulators) is clear before the first product
    asm volatile("bar.sync 4, %0;" ::"n"(128 * NW + 32) : "memory");
    tc_fence_after();
    for (int e = 0; e < ne + NB - 1; ++e) {
      if (e < ne) {
        const int st = e % RK, from = len - (last - e) * KT;
        const uint32_t tS = tmem + NC * (e % NB);
        mbar_wait_warp(bars.kfull + 8 * st, (e / RK) & 1, ctl, &g_tree_status, kErrWaitTma);
        if (from < KT) {
          zero_rows(smem + F::kBuf + F::kOne * st, KT, from, SUB);
          fence_async_smem();
          __syncwarp();
        }
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(lead, tS, dQ, (F::kBufSub >> 4) * s + 8 * F::kRows * (G - 1 - g) + 2 * kk, dK,
                     (F::kOne >> 4) * st + 8 * KT * s + 8 * NC * g + 2 * kk, id_s, g > 0 || s > 0 || kk > 0);
        mma_commit(lead, bars.sdone + 8 * (e % NB));
        mma_commit(lead, bars.kfree + 8 * st);
      }
      if (e >= NB - 1) {                                         // tile e - NB + 1 has been read: its buffer is next
        const int y = e - NB + 1, w = y % NW, st = y % RV;
        mbar_wait_warp(bars.ready + 8 * (y % NB), (y / NB) & 1, ctl, &g_tree_status, kErrWaitTile);
        tc_fence_after();
        if (OUT) {
          mbar_wait_warp(bars.vfull + 8 * st, (y / RV) & 1, ctl, &g_tree_status, kErrWaitTma);
          const int from = len - (last - y) * KT;
          if (from < KT) {
            zero_rows(smem + F::kBuf + F::kOne * (RK + st), KT, from, SUB);
            fence_async_smem();
            __syncwarp();
          }
          tc_fence_after();
          const uint32_t tP = tmem + NC * NB + F::kWgCols * w;
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int kk = 0; kk < NC / 16; ++kk)               // 16 keys per instruction: 16 rows of 128 B = 128 units
              mma_ts(lead, tP + 64, tP + (NC / 2) * g + 8 * kk, dV, (F::kOne >> 4) * st + 8 * NC * g + 128 * kk, id_p, 1);
          mma_commit(lead, bars.vfree + 8 * st);
          mma_commit(lead, bars.used + 8 * w);
        }
      }
    }
    mma_commit(lead, bars.alldone);
    __syncwarp();
  } else if (warp_u == 4 * NW + 1) {
    stream_tiles<D, KT, RK, RV, NB, OUT>(bars, &map_k, &map_v, ring_k, ring_v, last, -1, ne, nk, lead);
  } else {
    // ------------------------------------------------------------ the compute warps: lane = row of a group
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tP = tmem + NC * NB + F::kWgCols * wg + lanes, tO = tP + 64;
    const int g = row / F::kRows, x = row % F::kRows, r = r0 + x, rs = min(r, rows - 1);
    if (OUT) {
      uint32_t z[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) z[c] = 0u;
#pragma unroll
      for (int c = 0; c < 4 + D / 16; ++c) tmem_st16(tP + 16 * c, z);
      tmem_st_wait();
    }
    tc_fence_before();
    asm volatile("bar.sync 4, %0;" ::"n"(128 * NW + 32) : "memory");
    const bool cap = a.cap > 0.f;
    const float lin = cap ? a.cap * kLog2e : a.scale * kLog2e, pre = cap ? a.scale / a.cap : 0.f;
    float slope2 = 0.f;
    int at = len;
    if (a.slopes != nullptr) {
      slope2 = a.slopes[hk * a.group + rs / a.nodes] * kLog2e;
      at += lineage.depth[rs % a.nodes];
    }
    float ref = -INFINITY, s = 0.f;
    for (int e = wg; e < ne; e += NW) {
      const int j0 = (last - e) * KT + NC * g;
      mbar_wait_warp(bars.sdone + 8 * (e % NB), (e / NB) & 1, ctl, &g_tree_status, kErrWaitMma);
      // the product of the warpgroup's last tile has read its P~
      if (OUT && e >= NW) mbar_wait_warp(bars.used + 8 * wg, (e / NW - 1) & 1, ctl, &g_tree_status, kErrWaitMma);
      tc_fence_after();
      scan_step<D, NC, OUT>(tmem + NC * (e % NB) + lanes, tP + (NC / 2) * g, tO, lin, pre, cap, slope2, (float)(at - j0), len - j0, ref, s);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars.ready + 8 * (e % NB));
    }
    // rows that are laid out several times, and the warpgroups' keys, are one row
    sStat[wg * 128 + row] = make_float2(ref, s);
    float* sO = reinterpret_cast<float*>(smem + F::kBuf);           // [NW][128][D], over the ring
    if (OUT) {
      mbar_wait_warp(bars.alldone, 0, ctl, &g_tree_status, kErrWaitMma);
      tc_fence_after();
      __syncwarp();
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        float o[32];
        tmem_ld32(tO + c0, o);
        tmem_ld_wait(o);
        float4* dst = reinterpret_cast<float4*>(sO + (wg * 128 + row) * D + c0);
#pragma unroll
        for (int c = 0; c < 8; ++c) dst[c ^ (row & 7)] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(128 * NW) : "memory");
    constexpr int kUnits = OUT ? D / 4 : 1;
    const int64_t base = ((int64_t)nk * a.chunks + blockIdx.x) * rows;
    for (int y = tid; y < F::kRows * kUnits; y += 128 * NW) {
      const int xr = y / kUnits, c = y % kUnits;
      if (r0 + xr >= rows) break;
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int p = 0; p < NW * G; ++p) m = fmaxf(m, sStat[(p / G) * 128 + (p % G) * F::kRows + xr].x);
      const float from = m == -INFINITY ? 0.f : m;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < NW * G; ++p) {
        const int lane_row = (p / G) * 128 + (p % G) * F::kRows + xr;
        const float2 st = sStat[lane_row];
        const float f = fast_exp2(st.x - from);
        sum = fmaf(st.y, f, sum);
        if (OUT) {
          const float4 z = reinterpret_cast<const float4*>(sO + lane_row * D)[(c & ~7) | ((c & 7) ^ (lane_row & 7))];
          o.x = fmaf(z.x, f, o.x);
          o.y = fmaf(z.y, f, o.y);
          o.z = fmaf(z.z, f, o.z);
          o.w = fmaf(z.w, f, o.w);
        }
      }
      if (c == 0) a.part[base + r0 + xr] = make_float2(m, sum);
      if (OUT) reinterpret_cast<float4*>(a.pout + (base + r0 + xr) * D)[c] = o;
    }
  }
  drain_if_aborted(ctl);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free(tmem, F::kTmem);
}

// ---- sweep ---------------------------------------------------------------------------------------------
// What the thread of a key has to know of an accepted row: its lse, its position and the slope of its head.
struct RowStep {
  float lse;
  int at;
  float slope2;
  int pad;
};
// And of a draft's nodes, in their order: their lse (+inf behind the last: no bids), their parents; as bits, those that follow
// none (roots) or another than the one in front (far), and those whose demand such a later one starts from (keeps).
struct Walk {
  float lse[64];
  uint8_t up[64];
  uint32_t roots[2], far[2], keeps[2];
};
// Threads 0 .. N - 1, each with its node's lse.
template <int N> __device__ __forceinline__ void keep_walk(Walk* w, const tree::Lineage& lineage, int nodes, float lse) {
  const int x = threadIdx.x, up = x < nodes ? lineage.parent[x] : -1;
  bool keep = false;
  if (x < nodes)
    for (int y = x + 2; y < nodes; ++y) keep = keep || lineage.parent[y] == x;
  w->lse[x] = x < nodes ? lse : INFINITY;
  w->up[x] = (uint8_t)max(up, 0);
  const unsigned active = N < 32 ? (1u << N) - 1 : 0xffffffffu;
  const unsigned root = __ballot_sync(active, up < 0), far = __ballot_sync(active, up >= 0 && up != x - 1), k = __ballot_sync(active, keep);
  if ((x & 31) == 0) {
    w->roots[x >> 5] = root;
    w->far[x >> 5] = far;
    w->keeps[x >> 5] = k;
  }
}

// Shares of one key (of this lane), whose scores by `rows` nodes are at tS and whose cached demand is base: bf16, the values' type, into
// row `row` of the [128][64] tile dst (their sum is of the rounded ones).  Eight nodes at a time, whose bids and shares have nothing to wait for; their demand is one chain.
// 256 heads of 64, 24 nodes over 16384 keys, us: 169; 16 at a time, each looked up in shared memory 222; one node 157.
template <int N>
__device__ __forceinline__ void share_keys(uint32_t tS, int rows, float lin, float eps, float base, bool live, const Walk& walk,
                                           uint8_t* dst, int row) {
  float left = base;
#pragma unroll
  for (int c0 = 0; c0 < N; c0 += 16) {
    if (c0 >= rows) break;
    float v[16];
    __syncwarp();
    tmem_ld16(tS + c0, v);
    tmem_ld_wait16(v);
    const uint32_t roots = walk.roots[c0 / 32] >> (c0 & 31), far = walk.far[c0 / 32] >> (c0 & 31), keeps = walk.keeps[c0 / 32] >> (c0 & 31);
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
      if (c0 + h >= rows) break;
      const float4 l0 = reinterpret_cast<const float4*>(walk.lse + c0 + h)[0], l1 = reinterpret_cast<const float4*>(walk.lse + c0 + h)[1];
      const uint2 ups = *reinterpret_cast<const uint2*>(walk.up + c0 + h);
      const float lse[8] = {l0.x, l0.y, l0.z, l0.w, l1.x, l1.y, l1.z, l1.w};
      float p[8], d[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        p[y] = fast_exp2(fmaf(v[h + y], lin, -lse[y]));
        if (!live) p[y] = 0.f;
      }
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        if (roots >> (h + y) & 1) left = base;
        if (far >> (h + y) & 1) {
          tmem_st_wait();
          tmem_ld1(tS + ((y < 4 ? ups.x : ups.y) >> (8 * (y & 3)) & 255), &left);
          tmem_ld_wait1(&left);
        }
        d[y] = left = left + p[y];
        if (keeps >> (h + y) & 1) tmem_st1(tS + c0 + h + y, left);
      }
      uint32_t w[4];
#pragma unroll
      for (int y = 0; y < 8; y += 2) w[y >> 1] = pack_pair(p[y] * fast_rcp(d[y] + eps), p[y + 1] * fast_rcp(d[y + 1] + eps));
      *reinterpret_cast<uint4*>(dst + swizzled(row, (c0 + h) / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  tmem_st_wait();
  fence_async_smem();
}

template <int D, int N, bool DILUTE> struct Sweep {
  static constexpr int kKeys = 128, kThreads = 320;
  static constexpr uint32_t kOne = 128 * D * 2;
  static constexpr int kSpace = D == 64 || !DILUTE ? 65536 : 131072, kStages = (int)(kSpace / kOne);
  static constexpr int kK = DILUTE ? kStages / 2 : kStages, kV = DILUTE ? kStages / 2 : 4;
  static constexpr uint32_t kQSub = N * 128;
  static constexpr int kQ = N * 128 * (D / 64), kRingBytes = (int)kOne * kStages;
  // Q | ring | share [2][128][64] | ones [2][16][64] | node steps and positions | barriers + control
  static constexpr int kShare = DILUTE ? 2 * 16384 : 0, kOnes = DILUTE ? 4096 : 0;
  static constexpr int kBytes = (kQ + 1023) / 1024 * 1024 + kRingBytes + kShare + kOnes + 64 * 16 + 256 + 512 + 1024;
  static constexpr int kBuffers = DILUTE ? 2 : 4, kTmem = 256;             // S^T [buffers] x 64, out^T 64, sums 64
  static constexpr int kPerSm = ctas_per_sm(kBytes, kTmem);
  static_assert(kK >= 2 && kBytes <= 231000, "shared memory");
};

// DILUTE: shares of the nodes and their part of share V.  Otherwise: advanced = committed + the bids of the accepted rows.
// grid = (chunks, 1, batch * kv_heads); N >= rows
template <int D, int N, bool DILUTE>
__global__ void __launch_bounds__(320, Sweep<D, N, DILUTE>::kPerSm) sweep_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                       const __grid_constant__ tree::Args a, const __grid_constant__ tree::Accept acc) {
  using F = Sweep<D, N, DILUTE>;
  constexpr int RK = F::kK, RV = F::kV, NB = F::kBuffers, KT = 128, SUB = D / 64, kQ = (F::kQ + 1023) / 1024 * 1024;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t *pShare = smem + kQ + F::kRingBytes, *pOnes = pShare + F::kShare;
  const uint32_t sQ = smem_u32(smem), ring_k = sQ + kQ, ring_v = ring_k + F::kOne * RK, sShare = smem_u32(pShare), sOnes = smem_u32(pOnes);
  RowStep* step = reinterpret_cast<RowStep*>(pOnes + F::kOnes);
  Walk* walk = reinterpret_cast<Walk*>(step);
  const StreamBars<RK, RV, NB> bars(reinterpret_cast<uint64_t*>(step + 64));
  Ctl* ctl = bars.ctl;
  __shared__ tree::Lineage lineage;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = tid >> 7, row = tid & 127;
  const int warp_u = uniform_warp();
  const uint32_t lead = elect_one();
  const int nk = blockIdx.z, b = nk / a.kv_heads, hk = nk % a.kv_heads;
  const int rows = DILUTE ? a.nodes : a.group * acc.accepted;
  const int len = (int)uniform(tree::cache_len(a.pos_dev, a.len, a.capacity));
  const int2 keys = tree::chunk_keys(len, a.chunks, blockIdx.x, KT);
  const int ne = (keys.y - keys.x + KT - 1) / KT, last = keys.x / KT + ne - 1;

  let_next_in();
  if (tid == 0) bars.init();
  tree::make_lineage(&lineage, a.parents + b * a.parent_stride, a.nodes);
  // row r of the sweep is row q_row(r) of the key head's queries
  auto q_row = [&](int r) { return DILUTE ? r : r / acc.accepted * a.nodes + tree::path_node(a, acc, b, r % acc.accepted); };
  for (int x = tid; x < N * 8 * SUB; x += F::kThreads) {
    const int sub = x / (N * 8), r = x / 8 % N, c = x % 8;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < rows)
      w = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + ((int64_t)nk * a.group * a.nodes + q_row(r)) * D +
                                          64 * sub + 8 * c);
    *reinterpret_cast<uint4*>(smem + sub * F::kQSub + swizzled(r, c)) = w;
  }
  if (DILUTE) {
    // shares of nodes behind the last stay zero; ones: column 0 of both groups of 64
    for (int x = tid; x < F::kShare / 16; x += F::kThreads) reinterpret_cast<uint4*>(pShare)[x] = make_uint4(0, 0, 0, 0);
    for (int x = tid; x < 256; x += F::kThreads)
      *reinterpret_cast<uint4*>(pOnes + (x >> 7) * 2048 + swizzled((x >> 3) & 15, x & 7)) = make_uint4((x & 7) == 0 ? 0x3f80u : 0u, 0u, 0u, 0u);
  }
  fence_async_smem();
  __syncwarp();
  if (warp == 0) tmem_alloc(smem_u32(&ctl->tmem), F::kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl->tmem);

  if (warp_u == 8) {
    // ------------------------------------------------------------ the warp that issues MMAs
    constexpr uint32_t id_s = instr_desc(128, N, 0, 0), id_o = instr_desc(128, N, 1, 1);
    const Desc dK = make_desc(ring_k, 16, 1024), dQ = make_desc(sQ, 16, 1024);
    const Desc dOnes = make_desc(sOnes, 2048, 1024);
    for (int e = 0; e < ne + NB - 1; ++e) {
      if (e < ne) {
        const int st = e % RK, from = len - (last - e) * KT;
        const uint32_t tS = tmem + 64 * (e % NB);
        mbar_wait_warp(bars.kfull + 8 * st, (e / RK) & 1, ctl, &g_tree_status, kErrWaitTma);
        if (from < KT) {
          zero_rows(smem + kQ + F::kOne * st, KT, from, SUB);
          fence_async_smem();
          __syncwarp();
        }
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ss(lead, tS, dK, (F::kOne >> 4) * st + 8 * KT * s + 2 * kk, dQ, (F::kQSub >> 4) * s + 2 * kk, id_s, s > 0 || kk > 0);
        mma_commit(lead, bars.sdone + 8 * (e % NB));
        mma_commit(lead, bars.kfree + 8 * st);
      }
      if (e >= NB - 1) {
        const int y = e - NB + 1, w = y & 1, st = y % RV;
        mbar_wait_warp(bars.ready + 8 * (y % NB), (y / NB) & 1, ctl, &g_tree_status, kErrWaitTile);
        tc_fence_after();
        if (DILUTE) {
          mbar_wait_warp(bars.vfull + 8 * st, (y / RV) & 1, ctl, &g_tree_status, kErrWaitTma);
          const int from = len - (last - y) * KT;
          if (from < KT) {
            zero_rows(smem + kQ + F::kOne * (RK + st), KT, from, SUB);
            fence_async_smem();
            __syncwarp();
          }
          tc_fence_after();
          const uint32_t v = ring_v + F::kOne * st;
          const Desc dP = make_desc(sShare + 16384 * w, 16384, 1024);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            // heads of 64: the second 64 rows of A are the ones, out^T has the sums in row 64
            const uint32_t at = v + 2048 * kk;
            mma_ss(lead, tmem + 64 * NB, make_desc(at, D == 64 ? sOnes - at : KT * 128, 1024), 0, dP, 128 * kk, id_o, y > 0 || kk > 0);
            if (D == 128) mma_ss(lead, tmem + 64 * NB + 64, dOnes, 0, dP, 128 * kk, id_o, y > 0 || kk > 0);
          }
          mma_commit(lead, bars.vfree + 8 * st);
          mma_commit(lead, bars.used + 8 * w);
        }
      }
    }
    mma_commit(lead, bars.alldone);
    __syncwarp();
  } else if (warp_u == 9) {
    stream_tiles<D, KT, RK, RV, NB, DILUTE>(bars, &map_k, &map_v, ring_k, ring_v, last, -1, ne, nk, lead);
  } else {
    // ------------------------------------------------------------ the compute warps: lane = key
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const bool cap = a.cap > 0.f;
    const float lin = cap ? a.cap * kLog2e : a.scale * kLog2e, pre = cap ? a.scale / a.cap : 0.f;
    // what the keys' threads have to know of the rows; their lse may come from a kernel that has not ended yet
    if (DILUTE) wait_for_last();
    if (tid < N) {
      RowStep s{0.f, 0, 0.f, 0};
      const int q = tid < rows ? q_row(tid) : 0;
      if (tid < rows) s.lse = a.lse[((int64_t)nk * a.group) * a.nodes + q];
      if (DILUTE) {
        keep_walk<N>(walk, lineage, rows, s.lse);
      } else {
        if (tid < rows) {
          s.slope2 = a.slopes != nullptr ? a.slopes[hk * a.group + q / a.nodes] * kLog2e : 0.f;
          s.at = len + lineage.depth[q % a.nodes];
        }
        step[tid] = s;
      }
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    // (a key's demand is asked for a turn ahead)
    auto demand = [&](int e) {
      const int j = (last - e) * KT + row;
      return e < ne && j < len ? a.committed[(int64_t)nk * a.capacity + j] : 0.f;
    };
    float next = demand(wg);
    for (int e = wg; e < ne; e += 2) {
      const int j = (last - e) * KT + row;
      const bool live = j < len;
      const int64_t at = (int64_t)nk * a.capacity + j;
      const float base = next;
      next = demand(e + 2);
      const uint32_t tS = tmem + 64 * (e % NB) + lanes;
      mbar_wait_warp(bars.sdone + 8 * (e % NB), (e / NB) & 1, ctl, &g_tree_status, kErrWaitMma);
      // the product of the warpgroup's last tile has read its shares
      if (DILUTE && e >= 2) mbar_wait_warp(bars.used + 8 * wg, (e / 2 - 1) & 1, ctl, &g_tree_status, kErrWaitMma);
      tc_fence_after();
      if (DILUTE) {
        share_keys<N>(tS, rows, lin, a.eps, base, live, *walk, pShare + 16384 * wg, row);
      } else {
        float total = base;
#pragma unroll
        for (int c0 = 0; c0 < N; c0 += 16) {
          if (c0 >= rows) break;
          float v[16];
          __syncwarp();
          tmem_ld16(tS + c0, v);
          tmem_ld_wait16(v);
          if (cap) cap_scores<16>(v, pre, lin > kWideCap * kLog2e);
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const RowStep s = step[c0 + y];
            const float z = fmaf(v[y], lin, -s.lse - s.slope2 * (float)(s.at - j));
            if (c0 + y < rows) total += fast_exp2(z);
          }
        }
        if (live) acc.advanced[at] = total;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars.ready + 8 * (e % NB));
    }
    mbar_wait_warp(bars.alldone, 0, ctl, &g_tree_status, kErrWaitMma);
    tc_fence_after();
    if (DILUTE && wg == 0) {
      // out^T: lane = feature.  Chunks without keys have no product to read.
      const int64_t first_row = ((int64_t)nk * a.chunks + blockIdx.x) * rows;
#pragma unroll
      for (int c0 = 0; c0 < N; c0 += 16) {
        float o[16], t[16];
        __syncwarp();
        tmem_ld16(tmem + 64 * NB + lanes + c0, o);
        tmem_ld_wait16(o);
        if (D == 128) {
          tmem_ld16(tmem + 64 * NB + 64 + lanes + c0, t);
          tmem_ld_wait16(t);
        }
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          if (c0 + y >= rows) break;
          if (row < D) a.pout[(first_row + c0 + y) * D + row] = ne > 0 ? o[y] : 0.f;
          if (row == (D == 64 ? 64 : 0)) a.psum[first_row + c0 + y] = ne > 0 ? (D == 64 ? o[y] : t[y]) : 0.f;
        }
      }
    }
  }
  drain_if_aborted(ctl);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free(tmem, F::kTmem);
}

// ---- a dilution layer's step by clusters -----------------------------------------------------------------
// scan_kernel and sweep_kernel one after the other, for a head per cluster of eight CTAs: each reads its chunk of keys twice, the
// second time out of L2; statistics and outputs are joined through distributed shared memory.  The nodes' own keys are dealt out to
// the CTAs like cached ones.  One launch for the four of a step in chunks (trees.cu has the sizes it is taken for).
constexpr int kDraftRanks = 8;
template <int D, int N> struct Draft {
  static constexpr int kThreads = 320, G = N == 64 ? 2 : 4, kRows = 128 / G, kKeysA = 32 * G;
  static constexpr uint32_t kOneA = kKeysA * D * 2, kOne = 128 * D * 2;
  static constexpr int kSpace = D == 64 ? 65536 : 131072, RA = kSpace / (int)kOneA, R = kSpace / (int)kOne / 2, NA = 4, NB = 2;
  static constexpr int kBufRows = (G - 1) * kRows + 128;
  static constexpr uint32_t kBufSub = kBufRows * 128, kQSub = N * 128;
  static constexpr int kBuf = (int)kBufSub * (D / 64), kQ = (N * 128 * (D / 64) + 1023) / 1024 * 1024;
  static constexpr int kShare = 2 * 16384, kOnes = D == 64 ? 2048 : 4096, kOver = kBuf > kShare + kOnes ? kBuf : kShare + kOnes;
  static constexpr int kCols = N / kDraftRanks;                          // nodes' keys of a CTA
  // Q | ring | first the rows between zeros, then shares and ones | z [N][kCols] | steps | statistics of the rows | barriers
  static constexpr int kZ = N * kCols * 4;
  static constexpr int kBytes = kQ + kSpace + kOver + kZ + 64 * 16 + 64 * 8 + 640 + 1024;
  static constexpr int kTmem = 256, kPerSm = ctas_per_sm(kBytes, kTmem);
  static_assert(StreamBars<RA, 4, NA>::kBytes + StreamBars<R, R, NB>::kBytes + 16 <= 640 && kBytes <= 231000, "shared memory");
  static_assert(N * D * 4 + 256 <= kSpace, "a chunk's output fits the ring");
};

// grid = heads * 8, clusters of 8
template <int D, int N>
__global__ void __launch_bounds__(320, Draft<D, N>::kPerSm) draft_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v,
                                                                      const __grid_constant__ tree::Args a) {
  using F = Draft<D, N>;
  constexpr int SUB = D / 64, G = F::G, KA = F::kKeysA, RA = F::RA, NA = F::NA, R = F::R, NB = F::NB, C = kDraftRanks;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t *pRing = smem + F::kQ, *pOver = pRing + F::kSpace, *pShare = pOver, *pOnes = pOver + F::kShare;
  const uint32_t sQ = smem_u32(smem), ring = smem_u32(pRing), ring_v = ring + F::kOne * R, sOver = smem_u32(pOver), sOnes = smem_u32(pOnes);
  float* z = reinterpret_cast<float*>(pOver + F::kOver);                                   // [N][kCols]
  Walk* walk = reinterpret_cast<Walk*>(z + N * F::kCols);
  float2* chunk = reinterpret_cast<float2*>(z + N * F::kCols + 256);                                    // [N] this CTA's (maximum, sum)
  uint64_t* at_bars = reinterpret_cast<uint64_t*>(chunk + 64);
  const StreamBars<RA, 4, NA> ba(at_bars + 2);
  const StreamBars<R, R, NB> bb(at_bars + 2 + StreamBars<RA, 4, NA>::kBytes / 8);
  Ctl* ctl = ba.ctl;
  __shared__ tree::Lineage lineage;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = tid >> 7, row = tid & 127;
  const int warp_u = uniform_warp();
  const uint32_t lead = elect_one();
  const int rank = blockIdx.x % C, nk = blockIdx.x / C, n = a.nodes;
  const int len = (int)uniform(tree::cache_len(a.pos_dev, a.len, a.capacity));
  const int2 keys = tree::chunk_keys(len, C, rank, 128);
  const int na = (keys.y - keys.x + KA - 1) / KA, last = keys.x / KA + na - 1, ne = (keys.y - keys.x + 127) / 128, first = keys.x / 128;

  if (tid == 0) {
    ba.init();
    bb.init();
  }
  auto load_row = [&](int r, int sub, int c) {
    return *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + ((int64_t)nk * n + r) * D + 64 * sub + 8 * c);
  };
  for (int x = tid; x < F::kBufRows * 8 * SUB; x += F::kThreads) {
    const int sub = x / (F::kBufRows * 8), br = x / 8 % F::kBufRows, c = x % 8, r = br - (G - 1) * F::kRows;
    *reinterpret_cast<uint4*>(pOver + sub * F::kBufSub + swizzled(br, c)) = r >= 0 && r < min(n, F::kRows) ? load_row(r, sub, c) : make_uint4(0, 0, 0, 0);
  }
  for (int x = tid; x < N * 8 * SUB; x += F::kThreads) {
    const int sub = x / (N * 8), r = x / 8 % N, c = x % 8;
    *reinterpret_cast<uint4*>(smem + sub * F::kQSub + swizzled(r, c)) = r < n ? load_row(r, sub, c) : make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  tree::make_lineage(&lineage, a.parents + nk / a.kv_heads * a.parent_stride, n);
  __syncwarp();
  if (warp == 0) tmem_alloc(smem_u32(&ctl->tmem), F::kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl->tmem);

  if (warp_u == 8) {
    // ------------------------------------------------------------ the warp that issues MMAs
    cluster_arrive();
    {
      constexpr uint32_t id_s = instr_desc(128, 32, 0, 0);
      const Desc dQ = make_desc(sOver, 16, 1024), dK = make_desc(ring, 16, 1024);
      for (int e = 0; e < na + NA - 1; ++e) {
        if (e < na) {
          const int st = e % RA, from = len - (last - e) * KA;
          mbar_wait_warp(ba.kfull + 8 * st, (e / RA) & 1, ctl, &g_tree_status, kErrWaitTma);
          if (from < KA) {
            zero_rows(pRing + F::kOneA * st, KA, from, SUB);
            fence_async_smem();
            __syncwarp();
          }
          tc_fence_after();
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int s = 0; s < SUB; ++s)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_ss(lead, tmem + 32 * (e % NA), dQ, (F::kBufSub >> 4) * s + 8 * F::kRows * (G - 1 - g) + 2 * kk, dK,
                       (F::kOneA >> 4) * st + 8 * KA * s + 8 * 32 * g + 2 * kk, id_s, g > 0 || s > 0 || kk > 0);
          mma_commit(lead, ba.sdone + 8 * (e % NA));
          mma_commit(lead, ba.kfree + 8 * st);
        }
        if (e >= NA - 1) {
          const int y = e - NA + 1;
          mbar_wait_warp(ba.ready + 8 * (y % NA), (y / NA) & 1, ctl, &g_tree_status, kErrWaitTile);
          tc_fence_after();
        }
      }
      mma_commit(lead, ba.alldone);
    }
    constexpr uint32_t id_s = instr_desc(128, N, 0, 0), id_o = instr_desc(128, N, 1, 1);
    const Desc dK = make_desc(ring, 16, 1024), dQ = make_desc(sQ, 16, 1024), dOnes = make_desc(sOnes, 2048, 1024);
    for (int e = 0; e < ne + NB - 1; ++e) {
      if (e < ne) {
        const int st = e % R, from = len - (first + e) * 128;
        mbar_wait_warp(bb.kfull + 8 * st, (e / R) & 1, ctl, &g_tree_status, kErrWaitTma);
        if (from < 128) {
          zero_rows(pRing + F::kOne * st, 128, from, SUB);
          fence_async_smem();
          __syncwarp();
        }
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ss(lead, tmem + 64 * (e % NB), dK, (F::kOne >> 4) * st + 8 * 128 * s + 2 * kk, dQ, (F::kQSub >> 4) * s + 2 * kk, id_s,
                   s > 0 || kk > 0);
        mma_commit(lead, bb.sdone + 8 * (e % NB));
        mma_commit(lead, bb.kfree + 8 * st);
      }
      if (e >= NB - 1) {
        const int y = e - NB + 1, w = y & 1, st = y % R;
        mbar_wait_warp(bb.ready + 8 * (y % NB), (y / NB) & 1, ctl, &g_tree_status, kErrWaitTile);
        mbar_wait_warp(bb.vfull + 8 * st, (y / R) & 1, ctl, &g_tree_status, kErrWaitTma);
        const int from = len - (first + y) * 128;
        if (from < 128) {
          zero_rows(pRing + F::kOne * (R + st), 128, from, SUB);
          fence_async_smem();
          __syncwarp();
        }
        tc_fence_after();
        const uint32_t v = ring_v + F::kOne * st;
        const Desc dP = make_desc(smem_u32(pShare) + 16384 * w, 16384, 1024);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t at = v + 2048 * kk;
          mma_ss(lead, tmem + 128, make_desc(at, D == 64 ? sOnes - at : 128 * 128, 1024), 0, dP, 128 * kk, id_o, y > 0 || kk > 0);
          if (D == 128) mma_ss(lead, tmem + 192, dOnes, 0, dP, 128 * kk, id_o, y > 0 || kk > 0);
        }
        mma_commit(lead, bb.vfree + 8 * st);
        mma_commit(lead, bb.used + 8 * w);
      }
    }
    mma_commit(lead, bb.alldone);
    __syncwarp();
    cluster_wait();
    cluster_sync();
  } else if (warp_u == 9) {
    cluster_arrive();
    stream_tiles<D, KA, RA, 4, NA, false>(ba, &map_k, &map_v, ring, ring, last, -1, na, nk, lead);
    // (every product has read the first pass's stages)
    mbar_wait_warp(ba.alldone, 0, ctl, &g_tree_status, kErrWaitMma);
    stream_tiles<D, 128, R, R, NB, true>(bb, &map_k, &map_v, ring, ring_v, first, 1, ne, nk, lead);
    cluster_wait();
    cluster_sync();
  } else {
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const float lin = a.scale * kLog2e;
    const int cols = (n - rank + C - 1) / C;                               // nodes rank, rank + 8, ..
    // scores of the nodes against this CTA's nodes, while the first tiles come
    for (int x = tid; x < n * cols; x += 256) {
      const int i = x / cols, c = x % cols, key = rank + C * c;
      float s = -INFINITY;
      if (lineage.line[i] >> key & 1) {
        const uint4* q = reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((int64_t)nk * n + i) * D);
        const uint4* k = reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.kn + ((int64_t)nk * n + key) * D);
        s = 0.f;
#pragma unroll 4
        for (int y = 0; y < D / 8; ++y) {
          const uint4 u = q[y], v = k[y];
          const __nv_bfloat16 *p = reinterpret_cast<const __nv_bfloat16*>(&u), *w = reinterpret_cast<const __nv_bfloat16*>(&v);
#pragma unroll
          for (int t = 0; t < 8; ++t) s = fmaf(to_f32(p[t]), to_f32(w[t]), s);
        }
        s *= lin;
      }
      z[i * F::kCols + c] = s;
    }
    // ---------------------------------------------------------- statistics: lane = row of a group
    float ref = -INFINITY, sum = 0.f;
    const int g = row / F::kRows;
    for (int e = wg; e < na; e += 2) {
      const int j0 = (last - e) * KA + 32 * g;
      mbar_wait_warp(ba.sdone + 8 * (e % NA), (e / NA) & 1, ctl, &g_tree_status, kErrWaitMma);
      tc_fence_after();
      scan_step<D, 32, false>(tmem + 32 * (e % NA) + lanes, 0, 0, lin, 0.f, false, 0.f, 0.f, len - j0, ref, sum);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ba.ready + 8 * (e % NA));
    }
    mbar_wait_warp(ba.alldone, 0, ctl, &g_tree_status, kErrWaitMma);
    tc_fence_after();
    float2* stat = reinterpret_cast<float2*>(pOver);                        // [2][128], over the rows between zeros
    stat[wg * 128 + row] = make_float2(ref, sum);
    asm volatile("bar.sync 2, 256;" ::: "memory");
    for (int x = warp; x < n; x += 8) {
      float2 p = make_float2(-INFINITY, 0.f);
      if (lane < 2 * G) p = stat[(lane / G) * 128 + (lane % G) * F::kRows + x];
      float m = warp_max(p.x);
      float s = warp_sum(lane < 2 * G ? p.y * fast_exp2(p.x - (m == -INFINITY ? 0.f : m)) : 0.f);
      if (!isfinite(s) || m == INFINITY) {
        const float2 again = tree::redo_stats<D>(a, nk, x, 0, 0.f, keys.x, keys.y);
        m = again.x;
        s = again.y;
      }
      const float own = lane < cols ? z[x * F::kCols + lane] : -INFINITY, top = fmaxf(m, warp_max(own)), from = top == -INFINITY ? 0.f : top;
      s = s * exp2f(m - from) + warp_sum(lane < cols ? exp2f(own - from) : 0.f);
      if (lane == 0) chunk[x] = make_float2(top, s);
    }
    cluster_sync();
    for (int x = tid; x < F::kShare / 16; x += 256) reinterpret_cast<uint4*>(pShare)[x] = make_uint4(0, 0, 0, 0);
    for (int x = tid; x < F::kOnes / 16; x += 256)
      *reinterpret_cast<uint4*>(pOnes + (x >> 7) * 2048 + swizzled((x >> 3) & 15, x & 7)) = make_uint4((x & 7) == 0 ? 0x3f80u : 0u, 0u, 0u, 0u);
    if (tid < N) {
      float lse = 0.f;
      if (tid < n) {
        float m[C], t[C], top = -INFINITY, all = 0.f;
#pragma unroll
        for (int y = 0; y < C; ++y) {
          m[y] = ld_cluster(&chunk[tid].x, y);
          t[y] = ld_cluster(&chunk[tid].y, y);
          top = fmaxf(top, m[y]);
        }
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int y = 0; y < C; ++y) all = fmaf(t[y], exp2f(m[y] - from), all);
        lse = from + log2f(all);
        if (rank == 0) a.lse[(int64_t)nk * n + tid] = lse;
      }
      keep_walk<N>(walk, lineage, n, lse);
    }
    fence_async_smem();
    asm volatile("bar.sync 2, 256;" ::: "memory");
    // ---------------------------------------------------------- shares: lane = key
    for (int e = wg; e < ne; e += 2) {
      const int j = (first + e) * 128 + row;
      const bool live = j < len;
      const float base = live ? a.committed[(int64_t)nk * a.capacity + j] : 0.f;
      mbar_wait_warp(bb.sdone + 8 * (e % NB), (e / NB) & 1, ctl, &g_tree_status, kErrWaitMma);
      if (e >= 2) mbar_wait_warp(bb.used + 8 * wg, (e / 2 - 1) & 1, ctl, &g_tree_status, kErrWaitMma);
      tc_fence_after();
      share_keys<N>(tmem + 64 * (e % NB) + lanes, n, lin, a.eps, base, live, *walk, pShare + 16384 * wg, row);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bb.ready + 8 * (e % NB));
    }
    mbar_wait_warp(bb.alldone, 0, ctl, &g_tree_status, kErrWaitMma);
    tc_fence_after();
    // the chunk's output [N][D] and sums of shares, over the ring
    float *out = reinterpret_cast<float*>(pRing), *total = out + N * D;
    if (wg == 0) {
#pragma unroll
      for (int c0 = 0; c0 < N; c0 += 16) {
        float o[16], t[16];
        __syncwarp();
        tmem_ld16(tmem + 128 + lanes + c0, o);
        tmem_ld_wait16(o);
        if (D == 128) {
          tmem_ld16(tmem + 192 + lanes + c0, t);
          tmem_ld_wait16(t);
        }
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          if (row < D) out[(c0 + y) * D + row] = ne > 0 ? o[y] : 0.f;
          if (row == (D == 64 ? 64 : 0)) total[c0 + y] = ne > 0 ? (D == 64 ? o[y] : t[y]) : 0.f;
        }
      }
    } else if (row < cols) {
      // shares of this CTA's nodes' keys: the demand that a node leaves, then its share, in the place of its score
      const int key = rank + C * row;
      for (int x = 0; x < n; ++x) {
        float& cell = z[x * F::kCols + row];
        float left = 0.f;
        if (lineage.line[x] >> key & 1) left = exp2f(cell - walk->lse[x]) + (lineage.parent[x] >= 0 ? z[lineage.parent[x] * F::kCols + row] : 0.f);
        cell = left;
      }
      for (int x = n - 1; x >= 0; --x) {                 // (children come behind their parents)
        float& cell = z[x * F::kCols + row];
        const float had = lineage.parent[x] >= 0 ? z[lineage.parent[x] * F::kCols + row] : 0.f;
        cell = lineage.line[x] >> key & 1 ? (cell - had == 0.f ? 0.f : (cell - had) / (cell + a.eps)) : 0.f;
      }
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    for (int x = tid; x < n * D; x += 256) {
      const int i = x / D, d = x % D;
      float o = out[x], t = 0.f;
      for (int c = 0; c < cols; ++c) {
        const float w = z[i * F::kCols + c];
        t += w;
        if (w != 0.f) o = fmaf(w, to_f32(((const __nv_bfloat16*)a.vn)[((int64_t)nk * n + rank + C * c) * D + d]), o);
      }
      out[x] = o;
      if (d == 0) total[i] += t;
    }
    cluster_sync();
    for (int x = tid; x < (n - rank + C - 1) / C * D; x += 256) {
      const int i = rank + C * (x / D), d = x % D;
      float o = 0.f, t = 0.f;
#pragma unroll
      for (int y = 0; y < C; ++y) {
        o += ld_cluster(out + i * D + d, y);
        t += ld_cluster(total + i, y);
      }
      reinterpret_cast<__nv_bfloat16*>(a.out)[((int64_t)nk * n + i) * D + d] = from_f32<__nv_bfloat16>(o / (t + a.eps));
    }
  }
  drain_if_aborted(ctl);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free(tmem, F::kTmem);
  cluster_sync();                      // no CTA leaves while another may read its output
}

}  // namespace tc
}  // namespace dil
