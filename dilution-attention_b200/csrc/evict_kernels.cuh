// A cache's keys that were bid for least make room: of each (batch, head) row the first `sinks` keys, the last `recent`
// and, of those between, the ones of the highest rank stay, in their order.
//
// select_kernel finds the rank of the last key that stays, digit by digit of its bits (11, 11 and 10), each from one
// histogram of the row, and writes the positions that stay.  Ranks are compared as torch.sort does: NaN above every
// number, -0 like 0, equal ones by position.  A row's keys are spread over the CTAs of a cluster, which hold them in
// shared memory through the passes (rows too long for that read them again) and add up their histograms through
// distributed shared memory.  gather_kernel then moves the rows, and is bound by the bytes it moves.
#pragma once

#include "common.cuh"

namespace dil {
namespace evict {

constexpr int kThreads = 512;
constexpr int kBins = 2048;
constexpr int kMaxHeld = 48 * 1024;      // keys of a CTA that fit its shared memory (192 KB)

struct Args {
  const float* scores;       // (n, score_stride)
  int64_t score_stride;
  int length, keep, recent, sinks, seg;
  int held;                  // a CTA's keys fit its shared memory
  int* index;                // (n, keep)
};

// Bits that grow with the rank.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* p, int rank) {
  return __float_as_uint(ld_cluster(reinterpret_cast<const float*>(p), rank));
}

struct Shared {
  uint32_t hist[kBins];
  uint32_t warps[2][kThreads / 32];
  uint32_t counts[2];          // this CTA's: keys that stay whatever the ties, keys at the threshold
  uint32_t digit, need;
};

// Counts of a and b in front of the thread within the block, and the block's sums.  Two barriers.
__device__ __forceinline__ void block_counts(Shared& s, bool a, bool b, uint32_t& before_a, uint32_t& before_b, uint32_t& all_a,
                                             uint32_t& all_b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t ma = __ballot_sync(0xffffffffu, a), mb = __ballot_sync(0xffffffffu, b), below = (1u << lane) - 1;
  if (lane == 0) { s.warps[0][warp] = __popc(ma); s.warps[1][warp] = __popc(mb); }
  __syncthreads();
  before_a = __popc(ma & below);
  before_b = __popc(mb & below);
  all_a = all_b = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const uint32_t x = s.warps[0][w], y = s.warps[1][w];
    if (w < warp) { before_a += x; before_b += y; }
    all_a += x;
    all_b += y;
  }
  __syncthreads();
}

// grid = clusters of `ranks` CTAs, one per row.
__global__ void __launch_bounds__(kThreads) select_kernel(Args a, int ranks) {
  extern __shared__ uint32_t held[];
  __shared__ Shared s;
  const int tid = threadIdx.x, rank = blockIdx.x % ranks;
  const int64_t n = blockIdx.x / ranks;
  const float* scores = a.scores + n * a.score_stride;
  const int i0 = min(a.length, rank * a.seg), i1 = min(a.length, i0 + a.seg);
  const int c0 = a.sinks, c1 = a.length - a.recent;                 // the keys that have to prove themselves
  if (a.held) {
    for (int i = i0 + tid; i < i1; i += kThreads) held[i - i0] = rank_bits(scores[i]);
    __syncthreads();
  }
  auto bits = [&](int i) { return a.held ? held[i - i0] : rank_bits(scores[i]); };
  uint32_t need = a.keep - a.sinks - a.recent, prefix = 0, mask = 0;
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      for (int x = tid; x < kBins; x += kThreads) s.hist[x] = 0;
      __syncthreads();
      const int lo = max(i0, c0), hi = min(i1, c1);
      for (int base = lo; base < hi; base += kThreads) {
        const int i = base + tid;
        int d = -1;
        if (i < hi) {
          const uint32_t u = bits(i);
          if ((u & mask) == prefix) d = (u >> shift) & (bins - 1);
        }
        // a warp of one digit (fresh keys are alike) adds once
        if (__all_sync(0xffffffffu, d == __shfl_sync(0xffffffffu, d, 0))) {
          if ((tid & 31) == 0 && d >= 0) atomicAdd(&s.hist[d], 32u);
        } else if (d >= 0) {
          atomicAdd(&s.hist[d], 1u);
        }
      }
      if (ranks > 1) cluster_sync(); else __syncthreads();
      // thread t holds bins from the top: 4 t .. 4 t + 3 below the last
      uint32_t c[kBins / kThreads], sum = 0;
#pragma unroll
      for (int x = 0; x < kBins / kThreads; ++x) {
        const int bin = kBins - 1 - (tid * (kBins / kThreads) + x);
        c[x] = 0;
        if (ranks > 1)
          for (int y = 0; y < ranks; ++y) c[x] += ld_cluster_u32(&s.hist[bin], y);
        else c[x] = s.hist[bin];
        sum += c[x];
      }
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if ((tid & 31) >= o) inc += y;
      }
      if ((tid & 31) == 31) s.warps[0][tid >> 5] = inc;
      __syncthreads();
      uint32_t before = inc - sum;
      for (int w = 0; w < tid >> 5; ++w) before += s.warps[0][w];
      if (before < need && need <= before + sum) {
#pragma unroll
        for (int x = 0; x < kBins / kThreads; ++x) {
          if (before < need && need <= before + c[x]) {
            s.digit = kBins - 1 - (tid * (kBins / kThreads) + x);
            s.need = need - before;
          }
          before += c[x];
        }
      }
      if (ranks > 1) cluster_sync(); else __syncthreads();         // (the others have read this CTA's histogram too)
      prefix |= s.digit << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need = s.need;
      __syncthreads();
    }
  }
  // prefix is now the rank of the last key that stays, need how many of that rank do
  auto state = [&](int i, bool& above, bool& equal) {
    above = equal = false;
    if (i >= i1) return;
    if (i < c0 || i >= c1) { above = true; return; }
    const uint32_t u = bits(i);
    above = need > 0 && u > prefix;
    equal = need > 0 && u == prefix;
  };
  uint32_t above_before = 0, equal_before = 0;
  if (ranks > 1) {
    uint32_t na = 0, ne = 0;
    for (int i = i0 + tid; i < i1; i += kThreads) {
      bool above, equal;
      state(i, above, equal);
      na += above;
      ne += equal;
    }
    na = __reduce_add_sync(0xffffffffu, na);
    ne = __reduce_add_sync(0xffffffffu, ne);
    if (tid < 2) s.counts[tid] = 0;
    __syncthreads();
    if ((tid & 31) == 0) { atomicAdd(&s.counts[0], na); atomicAdd(&s.counts[1], ne); }
    cluster_sync();
    for (int y = 0; y < rank; ++y) {
      above_before += ld_cluster_u32(&s.counts[0], y);
      equal_before += ld_cluster_u32(&s.counts[1], y);
    }
  }
  int* index = a.index + n * a.keep;
  for (int base = i0; base < i1; base += kThreads) {
    bool above, equal;
    uint32_t xa, xe, ta, te;
    state(base + tid, above, equal);
    block_counts(s, above, equal, xa, xe, ta, te);
    xa += above_before;
    xe += equal_before;
    const uint32_t at = xa + min(xe, need);
    if ((above || (equal && xe < need)) && at < (uint32_t)a.keep) index[at] = base + tid;
    above_before += ta;
    equal_before += te;
  }
  if (ranks > 1) cluster_sync();        // no CTA leaves while another may read its counts
}

// Rows of k and v (16 bytes a thread) and their demand; zeros behind the last that stays.
__global__ void __launch_bounds__(256) gather_kernel(const uint4* __restrict__ k, const uint4* __restrict__ v,
                                                     const float* __restrict__ committed, const int* __restrict__ index,
                                                     int64_t n, int64_t capacity, int keep, int64_t new_capacity, int per,
                                                     uint4* __restrict__ k_out, uint4* __restrict__ v_out,
                                                     float* __restrict__ committed_out) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, place = at / per, row = place / new_capacity;
  if (row >= n) return;
  const int u = (int)(at % per);
  const int64_t x = place % new_capacity;
  uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
  float c = 0.f;
  if (x < keep) {
    const int64_t src = row * capacity + index[row * keep + x];
    kx = k[src * per + u];
    vx = v[src * per + u];
    if (u == 0 && committed != nullptr) c = committed[src];
  }
  k_out[at] = kx;
  v_out[at] = vx;
  if (u == 0 && committed != nullptr) committed_out[place] = c;
}

}  // namespace evict
}  // namespace dil
