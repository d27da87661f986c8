// A cache's keys that were bid for least make room: of each (batch, head) row the first `sinks` keys, the last `recent`
// and, of those between, the ones of the highest rank stay, in their order.
//
// select_kernel finds the rank of the last key that stays, eight bits at a time, each from one histogram of the row, and
// writes the positions that stay.  Ranks are compared as torch.sort does: NaN above every number, -0 like 0, equal ones by
// position.  A row's keys are spread over the CTAs of a cluster, which hold them in shared memory through the passes (rows
// too long for that read them again) and add up their histograms through distributed shared memory.  Where the clusters of
// all rows fill the chip, a cluster moves its row's keys itself, so that one row's passes, which wait for one another, run
// next to other rows' copies; few rows are moved by gather_kernel, on all SMs.  What bounds it are the bytes that are moved:
// 128 rows of 65536 keys, 16384 of which stay with heads of 64 in bf16, 236 us for 1.13 GB, 0.73 of the copy rate.
#pragma once

#include "common.cuh"

namespace dil {
namespace evict {

constexpr int kThreads = 512;
constexpr int kBins = 256;
constexpr int kCopies = 8;               // of a histogram: ranks share their first bits, and lanes that add to one word take turns
constexpr int kMaxHeld = 48 * 1024;      // keys of a CTA that fit its shared memory (192 KB)

struct Args {
  const float* scores;       // (n, score_stride)
  int64_t score_stride;
  int length, keep, recent, sinks, seg;
  int held;                  // a CTA's keys fit its shared memory
  int* index;                // (n, keep)
  const uint4* k;            // (n, capacity, 2^shift) units of 16 bytes
  const uint4* v;
  const float* committed;    // (n, capacity), or null
  int64_t capacity;
  int new_capacity, shift;
  int moves;                 // select_kernel moves the rows too
  uint4* k_out;              // (n, new_capacity, 2^shift)
  uint4* v_out;
  float* committed_out;
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

// Units [first, last) of a row's new places (2^shift units a key), N at a time a thread.
template <int THREADS, int N> __device__ __forceinline__ void move_units(const Args& a, int64_t row, int first, int last) {
  const int* index = a.index + row * a.keep;
  const uint4 *k_in = a.k + (row * a.capacity << a.shift), *v_in = a.v + (row * a.capacity << a.shift);
  const int64_t to = row * a.new_capacity;
  const int low = (1 << a.shift) - 1;
  auto position = [&](int at) {
    const int place = at >> a.shift;
    return at < last && place < a.keep ? __ldcg(index + place) : -1;
  };
  int src[N], next[N];               // (the next positions are under way while these rows are)
#pragma unroll
  for (int x = 0; x < N; ++x) next[x] = position(first + (int)threadIdx.x + x * THREADS);
  for (int base = first + (int)threadIdx.x; base < last; base += N * THREADS) {
    uint4 k[N], v[N];
#pragma unroll
    for (int x = 0; x < N; ++x) src[x] = next[x];
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int64_t from = ((int64_t)src[x] << a.shift) + (base + x * THREADS & low);
      k[x] = v[x] = make_uint4(0, 0, 0, 0);
      if (src[x] >= 0) {
        k[x] = __ldcs(k_in + from);
        v[x] = __ldcs(v_in + from);
      }
    }
#pragma unroll
    for (int x = 0; x < N; ++x) next[x] = position(base + (N + x) * THREADS);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int at = base + x * THREADS;
      if (at >= last) break;
      a.k_out[(to << a.shift) + at] = k[x];
      a.v_out[(to << a.shift) + at] = v[x];
      if ((at & low) == 0 && a.committed != nullptr)
        a.committed_out[to + (at >> a.shift)] = src[x] >= 0 ? a.committed[row * a.capacity + src[x]] : 0.f;
    }
  }
}

struct Shared {
  uint32_t copies[kBins * kCopies];
  uint32_t hist[2][kBins];     // the CTA's, two passes apart: the others may still read the last one
  uint32_t warps[2][kThreads / 32];
  uint32_t counts[2];          // this CTA's: keys that stay whatever the ties, keys at the threshold
  uint32_t digit, need, whole;
};

// grid = clusters of `ranks` CTAs, one per row.
__global__ void __launch_bounds__(kThreads, 4) select_kernel(Args a, int ranks) {
  extern __shared__ uint4 held4[];
  __shared__ Shared s;
  uint32_t* held = reinterpret_cast<uint32_t*>(held4);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x % ranks;
  const int64_t n = blockIdx.x / ranks;
  const float* scores = a.scores + n * a.score_stride;
  const int i0 = min(a.length, rank * a.seg), i1 = min(a.length, i0 + a.seg), count = i1 - i0;
  const int c0 = a.sinks - i0, c1 = a.length - a.recent - i0;       // the keys that have to prove themselves, from i0 on
  if (a.held) {
    for (int i = tid; i < count; i += kThreads) held[i] = rank_bits(scores[i0 + i]);
    __syncthreads();
  }
  auto bits = [&](int i) { return a.held ? held[i] : rank_bits(scores[i0 + i]); };
  uint32_t need = a.keep - a.sinks - a.recent, prefix = 0, mask = 0;
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      for (int x = tid; x < kBins * kCopies / 4; x += kThreads) reinterpret_cast<uint4*>(s.copies)[x] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      uint32_t* mine = s.copies + (tid & (kCopies - 1));
      const int lo = max(0, c0), hi = min(count, c1);
      auto add = [&](uint32_t u) {
        if ((u & mask) == prefix) atomicAdd(mine + (u >> shift & 255u) * kCopies, 1u);
      };
      if (a.held) {                  // four at a time; the first and the last four may be cut
        const int q0 = (lo + 3) / 4, q1 = max(q0, hi / 4);
        for (int q = q0 + tid; q < q1; q += kThreads) {
          const uint4 u = held4[q];
          add(u.x);
          add(u.y);
          add(u.z);
          add(u.w);
        }
        const int edge = tid < 4 ? lo + tid : 4 * q1 + tid - 4;
        if (tid < 8 && edge >= lo && edge < hi && (tid < 4 ? edge < 4 * q0 : true)) add(held[edge]);
      } else {
        for (int i = lo + tid; i < hi; i += kThreads) add(bits(i));
      }
      __syncthreads();
      if (tid < kBins) {
        const uint4 x = reinterpret_cast<const uint4*>(s.copies)[2 * tid], y = reinterpret_cast<const uint4*>(s.copies)[2 * tid + 1];
        s.hist[pass & 1][tid] = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
      }
      if (ranks > 1) cluster_sync(); else __syncthreads();
      // thread t < 256 holds bin 255 - t of the whole row
      uint32_t sum = 0;
      if (tid < kBins) {
        const uint32_t* bin = &s.hist[pass & 1][kBins - 1 - tid];
        if (ranks > 1) {
          uint32_t x[8];             // (all under way at once)
#pragma unroll
          for (int y = 0; y < 8; ++y) x[y] = y < ranks ? ld_cluster_u32(bin, y) : 0u;
#pragma unroll
          for (int y = 0; y < 8; ++y) sum += x[y];
        } else {
          sum = *bin;
        }
      }
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) s.warps[0][warp] = inc;
      __syncthreads();
      if (tid < kBins) {
        uint32_t before = inc - sum;
#pragma unroll
        for (int w = 0; w < kBins / 32; ++w) before += w < warp ? s.warps[0][w] : 0u;
        if (before < need && need <= before + sum) {
          s.digit = kBins - 1 - tid;
          s.need = need - before;
          s.whole = need == before + sum;
        }
      }
      __syncthreads();
      prefix |= s.digit << shift;
      mask |= 255u << shift;
      need = s.need;
      if (s.whole) break;              // every key of these bits stays: the others need not be told apart
    }
  }
  // prefix has the bits of the last key that stays, need is how many of those bits do
  auto state = [&](int i, bool& above, bool& equal) {
    above = equal = false;
    if (i >= count) return;
    if (i < c0 || i >= c1) { above = true; return; }
    if (need == 0) return;
    const uint32_t u = bits(i) & mask;
    above = u > prefix;
    equal = u == prefix;
  };
  // a warp has a stretch of its own: counts of the warps, then of the CTAs, then each walks through its stretch again
  constexpr int kWarps = kThreads / 32;
  const int per = ((count + kWarps - 1) / kWarps + 31) / 32 * 32, w0 = min(count, warp * per), w1 = min(count, w0 + per);
  uint32_t na = 0, ne = 0;
  for (int i = w0 + lane; i < w1; i += 32) {
    bool above, equal;
    state(i, above, equal);
    na += above;
    ne += equal;
  }
  na = __reduce_add_sync(0xffffffffu, na);
  ne = __reduce_add_sync(0xffffffffu, ne);
  if (lane == 0) { s.warps[0][warp] = na; s.warps[1][warp] = ne; }
  __syncthreads();
  uint32_t above_before = 0, equal_before = 0, all_above = 0, all_equal = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t x = s.warps[0][w], y = s.warps[1][w];
    if (w < warp) { above_before += x; equal_before += y; }
    all_above += x;
    all_equal += y;
  }
  if (ranks > 1) {
    if (tid == 0) { s.counts[0] = all_above; s.counts[1] = all_equal; }
    cluster_sync();
    for (int y = 0; y < rank; ++y) {
      above_before += ld_cluster_u32(&s.counts[0], y);
      equal_before += ld_cluster_u32(&s.counts[1], y);
    }
  }
  int* index = a.index + n * a.keep;
  const uint32_t below = (1u << lane) - 1;
  for (int base = w0; base < w1; base += 32) {
    bool above, equal;
    state(base + lane < w1 ? base + lane : count, above, equal);
    const uint32_t ma = __ballot_sync(0xffffffffu, above), me = __ballot_sync(0xffffffffu, equal);
    const uint32_t xe = equal_before + __popc(me & below), at = above_before + __popc(ma & below) + min(xe, need);
    if ((above || (equal && xe < need)) && at < (uint32_t)a.keep) index[at] = i0 + base + lane;
    above_before += __popc(ma);
    equal_before += __popc(me);
  }
  if (ranks > 1) cluster_sync(); else __syncthreads();        // (and no CTA leaves while another may read its counts)
  if (!a.moves) return;
  const int units = a.new_capacity << a.shift, part = (units + ranks - 1) / ranks;
  move_units<kThreads, 1>(a, n, min(units, rank * part), min(units, (rank + 1) * part));
}

// Rows of k and v and their demand; zeros behind the last that stays.  Four units of 16 bytes of each a thread.
__global__ void __launch_bounds__(256) gather_kernel(Args a) {
  const int units = a.new_capacity << a.shift, blocks = (units + 1023) / 1024, first = (int)(blockIdx.x % blocks) * 1024;
  move_units<256, 4>(a, blockIdx.x / blocks, first, min(units, first + 1024));
}

}  // namespace evict
}  // namespace dil
