// Softmax attention with caps, biases and masks (attend_common.cuh) on the tensor cores: bf16 heads of 64 and 128.
// Operand tiles come in by TMA, products are tcgen05.mma with accumulators in TMEM, and the values that a thread forms
// (P~, dS) go back into TMEM over the scores it has read, as the A operand of the next product: in bf16, the operands' type, each
// off by up to 2^-8 of itself.  References, sums, lse, delta and accumulators are fp32.  A warp of its own issues
// every copy and MMA.  Which pairs of tiles have anything to do is asked of the documents' ranges, never of a list.
//
//   forward : a CTA's query tile of 128 walks over half tiles of 64 keys; two warpgroups take them in turn.  lane = query:
//             reference, sums and accumulator of a row belong to one thread and warpgroup, and are merged once at the end.
//   backward: one kernel for both halves.  A tile of 128 stays (dq: queries with their dout; dk, dv: keys with their values),
//             half tiles of 64 of the other kind stream past; kWg warpgroups take them in turn, and accumulators in TMEM
//             are shared by all of them.  dq: lane = query.  dk, dv: lane = key, and nothing is reduced across CTAs: the heads
//             that share a key head stream past one after the other.  So scores are formed twice, seven products in
//             place of five, and no result depends on an order of atomic additions.
//
// What bounds them, per pair of tiles of 128 x 64: 512 cycles for one exponential a score on the special-function unit (16 a
// clock), and 256 (heads of 64: 128) cycles for each product on the tensor pipe, 8192 operations a clock: 2 forward, 4 for dk and dv, 3
// for dq.  So heads of 64 are bound by the exponentials forward and for dq and by both alike for dk and dv, heads of 128 by both
// alike forward and by the tensor pipe in the backward (1024 and 768 cycles).  Measured, forward / dk, dv / dq in us: n = 64, T = 8192,
// heads of 64 774 / 1079 / 896 (forward 0.62 of the exponentials' rate), documents of 700 tokens 231 / 246 / 196, where a block of
// a few half tiles is mostly its start and its end; n = 32 (8 key heads), T = 8192, heads of 128, capped 834 / 1030 / 840 (0.39 / 0.64 /
// 0.58 of the burst rate of a large bf16 product for the products that they take).
#pragma once

#include "attend_common.cuh"
#include "tc_score.cuh"

namespace dil {
namespace tc {

__device__ int g_attend_status = 0;        // first bounded wait that ran out (0 = none)

using attend::Row;

// ---- which pairs of tiles ------------------------------------------------------------------------
struct Docs {
  int lo, hi, id;          // smallest and largest id, and the one id of all tokens or -1
  bool holes;              // there is padding among them
};
__device__ __forceinline__ Docs docs_of(const Row& r, int i0, int i1) {
  Docs d{INT_MAX, -1, -1, false};
  bool pure = true;
  for (int s = i0 / attend::kSpan; s <= min(i1, r.t - 1) / attend::kSpan; ++s) {
    const attend::DocRange x = r.ranges[s];
    d.lo = min(d.lo, x.lo);
    d.hi = max(d.hi, x.hi);
    pure = pure && x.pure;
    d.holes = d.holes || x.holes;
  }
  if (pure && d.lo == d.hi) d.id = d.lo;
  return d;
}
// 0: no query of [i0, i1] sees a key of [j0, j1]; 2: each sees each; 1: masks decide (the kernels' lambdas: 3 where the half tile that
// passes has padding).  BIAS: distances of one sign only are
// left to the kernels' common path.  Rows behind the last token count as seen where they do no harm: queries, and keys
// of a tile that stays; j1 is the last key that matters then.
template <bool BIAS>
__device__ __forceinline__ int pair_state(const Row& r, int i0, int i1, const Docs& di, int j0, int j1, const Docs& dj) {
  if (j0 > i1 && j0 >= r.prefix) return 0;
  if (r.ranges != nullptr) {
    if (di.hi < dj.lo || dj.hi < di.lo) return 0;
    if (di.id < 0 || di.id != dj.id) return 1;
  }
  if (j1 >= r.t || (BIAS && j1 > i0)) return 1;
  return j1 <= i0 || j1 < r.prefix ? 2 : 1;
}

// ---- forward -----------------------------------------------------------------------------------------
// What pairs of tiles have to do is asked once per block and kept for this many half tiles from `base` on: two bits each, of 32
// half tiles in a word: the warp that issues MMAs has to know in a few cycles, it is what all others wait for.  masked: states 1 and
// 3; seen: states 1 and 2.
constexpr int kStates = 4096;
struct States {
  uint32_t seen[kStates / 32], masked[kStates / 32];
  __device__ __forceinline__ int of(int e) const { return masked[e / 32] >> (e & 31) & 1 ? 1 : (seen[e / 32] >> (e & 31) & 1) * 2; }
  __device__ __forceinline__ uint32_t any(int e) const { return seen[e / 32] | masked[e / 32]; }
  __device__ __forceinline__ uint32_t holes(int e) const { return masked[e / 32] & ~seen[e / 32]; }
};
// Half tiles [base, end); f: the state of one.  Returns the first and the last + 1 of the warp's that have anything to do.
template <typename F> __device__ __forceinline__ int2 keep_states(States* s, int base, int end, int warp, int warps, F f) {
  const int lane = threadIdx.x & 31;
  int2 range = make_int2(INT_MAX, 0);
  for (int e = base + 32 * warp; e < end; e += 32 * warps) {
    const int what = e + lane < end ? f(e + lane) : 0;
    const uint32_t any = __ballot_sync(0xffffffffu, what != 0), masked = __ballot_sync(0xffffffffu, what & 1);
    const uint32_t seen = __ballot_sync(0xffffffffu, what == 1 || what == 2);
    if (lane == 0 && e - base < kStates) {
      s->seen[(e - base) / 32] = seen;
      s->masked[(e - base) / 32] = masked;
    }
    if (any) range = make_int2(min(range.x, e + __ffs(any) - 1), e + 32 - __clz(any));
  }
  return range;
}
// The warps' ranges, put together by every warp.
__device__ __forceinline__ int2 all_of(const int2* range, int warps) {
  const int lane = threadIdx.x & 31;
  const int2 x = lane < warps ? range[lane] : make_int2(INT_MAX, 0);
  return make_int2((int)uniform(__reduce_min_sync(0xffffffffu, x.x)), (int)uniform(__reduce_max_sync(0xffffffffu, x.y)));
}

// Zeros for the padding among the 64 tokens (of `tokens` left) with ids docs, in their half tiles of SUB sub-tiles, two of them if `both`
// and that many bytes apart: what the values of padding are multiplied by is 0, which makes no number of those that are not
// finite.  One warp, in front of the half tile's products.
template <int SUB> __device__ __noinline__ void zero_holes(uint8_t* tile, uint32_t apart, bool both, const int* docs, int tokens) {
  const int lane = threadIdx.x & 31, id0 = lane < tokens ? docs[lane] : 0, id1 = lane + 32 < tokens ? docs[lane + 32] : 0;
  const uint32_t low = __ballot_sync(0xffffffffu, id0 < 0), high = __ballot_sync(0xffffffffu, id1 < 0);
#pragma unroll 4
  for (int x = lane; x < 64 * 8; x += 32) {              // 16 bytes of a row's 128 in a sub-tile
    const int row = x >> 3;
    if (!((row < 32 ? low : high) >> (row & 31) & 1)) continue;
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub) {
      uint8_t* at = tile + sub * (kTileBytes / 2) + 16 * x;
      *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
      if (both) *reinterpret_cast<uint4*>(at + apart) = make_uint4(0, 0, 0, 0);
    }
  }
  fence_async_smem();
  __syncwarp();
}

template <int D> struct AttendForward {
  static constexpr int kThreads = 256 + 32, kRing = 5;                              // half tiles of K and V
  static constexpr uint32_t kTile = Rows<kForm<D>>::kBytes, kHalf = kTile / 2;
  // Q | K[ring] | V[ring] | merge statistics [2][128] float2, float | flags [128] | barriers + control
  static constexpr int kOperands = (int)(kTile + 2 * kRing * kHalf);
  static constexpr int kStats = 2 * 128 * 12, kFlags = 128 * 4;
  static constexpr int kBytes = kOperands + kStats + kFlags + 256 + 1024;
  static constexpr int kBufs = D == 128 ? 2 : 1;                                   // score buffers of a warpgroup
  static constexpr int kWgCols = 64 * kBufs + D;
  static constexpr int kTmem = 2 * kWgCols <= 256 ? 256 : 512;
  static_assert(2 * kWgCols <= kTmem, "the warpgroups' columns fit the allocation");
  static_assert(128 * D * 4 <= (int)(2 * kRing * kHalf), "the merge area fits the ring");
};

constexpr float kAttendLimit = 1099511627776.f;      // 2^40: a half tile whose P~ sum to more moves the reference

// Bits of 64 tokens x0 .. that have the lane's document id, which may differ from lane to lane (a negative one: none).  Each lane
// brings two of the tokens' ids; lanes of one id are served together.
__device__ __forceinline__ uint2 document_bits(const Row& r, int x0, int id) {
  const int lane = threadIdx.x & 31, k0 = r.docs[min(x0 + lane, r.t - 1)], k1 = r.docs[min(x0 + 32 + lane, r.t - 1)];
  uint2 bits = make_uint2(0, 0);
  for (unsigned todo = __ballot_sync(0xffffffffu, id >= 0); todo;) {
    const int want = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
    const uint2 same = make_uint2(__ballot_sync(0xffffffffu, k0 == want), __ballot_sync(0xffffffffu, k1 == want));
    if (id == want) bits = same;
    todo &= ~__ballot_sync(0xffffffffu, id == want);
  }
  return bits;
}
// The lowest n of 64 bits.
__device__ __forceinline__ uint2 low_bits(int n) {
  return make_uint2(n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1, n >= 64 ? ~0u : n <= 32 ? 0u : (1u << (n - 32)) - 1);
}
__device__ __forceinline__ bool bit_of(const uint2& m, int e) { return (e < 32 ? m.x >> e : m.y >> (e - 32)) & 1; }
// Which of the keys j0 .. query i sees, and which of the queries i0 .. see key j.
__device__ __forceinline__ uint2 key_bits(const Row& r, int i, int j0) {
  uint2 m = low_bits(min(max(i + 1, r.prefix), r.t) - j0);
  if (r.docs != nullptr) {
    const uint2 d = document_bits(r, j0, r.docs[i]);
    m.x &= d.x;
    m.y &= d.y;
  }
  return m;
}
__device__ __forceinline__ uint2 query_bits(const Row& r, int i0, int j) {
  uint2 m = low_bits(r.t - i0);
  if (j >= r.prefix) {
    const uint2 x = low_bits(j - i0);
    m.x &= ~x.x;
    m.y &= ~x.y;
  }
  if (r.docs != nullptr) {
    const uint2 d = document_bits(r, i0, r.docs[j]);
    m.x &= d.x;
    m.y &= d.y;
  }
  return m;
}

// A warpgroup's step over the 64 scores of keys j0 .. at tS: P~ = 2^(z - reference) as bf16 over the scores, their sum into s, and that
// of the rounded ones, which out is divided by, into sr: the rounding of a P~ that a row is mostly made of then cancels (dq, dk of
// capped scores of deviation 3 against 64 bits by norm 0.0028 with one sum, 0.0025 with two; 767 -> 830 us at B2 H16 T8192 d128).
// The reference is the maximum of the first half tile that a row sees and moves where a later one's P~ sum to more than 2^40; only
// then is the accumulator rescaled, once its products are through (settled).  bf16 has the range of fp32: P~ below that limit
// keeps 8 bits.
template <int D, bool CAP, bool BIAS, typename Settled>
__device__ __forceinline__ void forward_step(uint32_t tS, uint32_t tO, const Row& r, float lin, float pre, int j0, int i, bool edge,
                                             float& ref, float& s, float& sr, Settled settled) {
  float v[64];
  uint32_t pw[32];
  float ps, pr;
  bool some = true;                  // the row sees any of the keys
  // the scores as z = mul v + add + step e, masked ones -inf
  auto fetch = [&]() {
    tmem_ld32(tS, v);
    tmem_ld32(tS + 32, v + 32);
    tmem_ld_wait(v);
    tmem_ld_wait(v + 32);
    if (CAP) cap_scores<64>(v, pre, r.cap2 > kWideCap * kLog2e);
    if (edge) {
      const uint2 m = key_bits(r, i, j0);
      some = (m.x | m.y) != 0;
      if (BIAS) {                    // distances of both signs
        const float far = (float)(i - j0);
#pragma unroll
        for (int e = 0; e < 64; ++e) v[e] = fmaf(v[e], lin, -r.slope2 * fabsf(far - (float)e));
      }
#pragma unroll
      for (int e = 0; e < 64; ++e) v[e] = bit_of(m, e) ? v[e] : -INFINITY;
    }
  };
  const float mul = BIAS && edge ? 1.f : lin, step = BIAS && !edge ? r.slope2 : 0.f;
  const float add = BIAS && !edge ? r.slope2 * (float)(j0 - i) : 0.f;
  auto exponentials = [&](float mul, float add, float step) {
    const float2 mm = make_float2(mul, mul), four = make_float2(4.f * step, 4.f * step);
    float2 a0 = make_float2(0.f, 0.f), b0 = a0;
    float2 o0 = make_float2(add, BIAS ? add + step : add), o1 = BIAS ? make_float2(add + 2.f * step, add + 3.f * step) : o0;
#pragma unroll
    for (int e = 0; e < 64; e += 4) {
      const float2 z0 = fma2(make_float2(v[e], v[e + 1]), mm, o0), z1 = fma2(make_float2(v[e + 2], v[e + 3]), mm, o1);
      if (BIAS) {
        o0 = add2(o0, four);
        o1 = add2(o1, four);
      }
      const float2 p0 = make_float2(fast_exp2(z0.x), fast_exp2(z0.y)), p1 = make_float2(fast_exp2(z1.x), fast_exp2(z1.y));
      a0 = add2(a0, add2(p0, p1));
      const uint32_t w0 = pack_pair(p0.x, p0.y), w1 = pack_pair(p1.x, p1.y);
      b0 = add2(b0, add2(unpack_pair(w0), unpack_pair(w1)));
      pw[e >> 1] = w0;
      pw[(e >> 1) + 1] = w1;
    }
    ps = a0.x + a0.y;
    pr = b0.x + b0.y;
  };
  fetch();
  bool slow = __any_sync(0xffffffffu, ref == -INFINITY && some);
  if (!slow) {
    exponentials(mul, ref == -INFINITY ? 0.f : add - ref, step);
    slow = __any_sync(0xffffffffu, !(ps < kAttendLimit));
    if (slow) fetch();               // rare: the scores are still in TMEM
  }
  if (slow) {
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 64; ++e) {
      v[e] = fmaf(v[e], mul, BIAS ? fmaf(step, (float)e, add) : 0.f);
      top = fmaxf(top, v[e]);
    }
    const float now = fmaxf(ref, top);
    if (__any_sync(0xffffffffu, now != ref)) {
      const bool fresh = __all_sync(0xffffffffu, ref == -INFINITY);        // nothing accumulated yet
      const float f = fast_exp2(ref - (now == -INFINITY ? 0.f : now));
      if (!fresh) {
        settled();
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
      sr *= f;
      ref = now;
    }
    exponentials(1.f, ref == -INFINITY ? 0.f : -ref, 0.f);
  }
  s += ps;
  sr += pr;
  tmem_st16(tS, pw);
  tmem_st16(tS + 16, pw + 16);
  tmem_st_wait();
}

// grid = batch * heads * ceil(t / 128), last queries (the longest rows) first.
template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(AttendForward<D>::kThreads, D == 64 ? 2 : 1) attend_forward_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
    const __grid_constant__ attend::Args a) {
  using F = AttendForward<D>;
  constexpr int W = kForm<D>, R = F::kRing;
  constexpr uint32_t TB = F::kTile, HB = F::kHalf, HSub = kTileBytes / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  const uint32_t sQ = smem_u32(smem), sK = sQ + TB, sV = sK + R * HB;
  float2* sStat = reinterpret_cast<float2*>(smem + F::kOperands);
  int* sFlag = reinterpret_cast<int*>(smem + F::kOperands + F::kStats);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::kOperands + F::kStats + F::kFlags);
  constexpr int NB = F::kBufs, NG = 2;                                        // score buffers, warpgroups
  const uint32_t qfull = smem_u32(bars), kfull = qfull + 8, kfree = kfull + 8 * R, sdone = kfree + 8 * R, odone = sdone + 8 * NB * NG,
                 pready = odone + 8 * NG;
  Ctl* ctl = reinterpret_cast<Ctl*>(bars + 1 + 2 * R + (2 * NB + 1) * NG);
  __shared__ int2 s_range[F::kThreads / 32];
  __shared__ States s_state;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = tid >> 7, row = tid & 127;
  const int warp_u = uniform_warp();
  const uint32_t lead = elect_one();
  const int heads = a.batch * a.heads, blocks = (a.t + kTileRows - 1) / kTileRows;
  const int n = (int)(blockIdx.x % heads), i0 = (blocks - 1 - (int)(blockIdx.x / heads)) * kTileRows;
  const int b = n / a.heads, h = n % a.heads, nk = b * a.kv_heads + h / (a.heads / a.kv_heads);
  const Row r = attend::make_row(a, b, h);
  const float lin = CAP ? r.cap2 : r.pre, pre = CAP ? a.scale / a.cap : 0.f;
  const Docs dq = r.ranges != nullptr ? docs_of(r, i0, i0 + kTileRows - 1) : Docs{INT_MAX, -1, -1, false};
  auto state = [&](int hh) {                            // of half tile hh
    const int j0 = hh * 64;
    const Docs dj = r.ranges != nullptr ? docs_of(r, j0, j0 + 63) : Docs{INT_MAX, -1, -1, false};
    const int what = pair_state<BIAS>(r, i0, i0 + kTileRows - 1, dq, j0, j0 + 63, dj);
    return what == 1 && dj.holes ? 3 : what;
  };

  const int top = (attend::key_end(r, min(r.t, i0 + kTileRows) - 1) + 63) / 64;
  if (tid == 0) {
    ctl->abort = 0;
    for (int x = 0; x < 1 + 2 * R + (NB + 1) * NG; ++x) mbar_init(qfull + 8 * x, 1);        // qfull, kfull, kfree, sdone, odone
    for (int x = 0; x < NB * NG; ++x) mbar_init(pready + 8 * x, 4);      // (of a buffer: a warp may be a half tile ahead of another)
    fence_barrier_init();
  }
  if (tid < 128) sFlag[tid] = 0;
  __syncwarp();
  if (warp == 0) tmem_alloc(smem_u32(&ctl->tmem), F::kTmem);
  const int2 mine = keep_states(&s_state, 0, top, warp, F::kThreads / 32, state);
  if (lane == 0) s_range[warp] = mine;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl->tmem);
  // half tiles [h0, h0 + nh) that any of the CTA's queries sees
  const int2 range = all_of(s_range, F::kThreads / 32);
  const int h0 = range.y > 0 ? range.x : 0, nh = range.y - h0;
  // nearest keys first: a distance bias has the largest scores there, and later half tiles do not move the reference
  const int last = h0 + nh - 1;

  if (warp_u == 8) {
    // ------------------------------------------------------------ the issuing warp
    constexpr uint32_t id_s = instr_desc(128, 64, 0, 0), id_p = instr_desc(128, D, 0, 1);
    const Desc dQ = make_desc(sQ, 16, 1024), dK = make_desc(sK, 16, 1024), dV = make_desc(sV, HSub, 1024);
    auto load_keys = [&](int e, int st) {
      if (!lead) return;
      mbar_expect_tx(kfull + 8 * st, 2 * HB);
      tma_load_rows<W>(sK + HB * st, &map_k, (last - e) * 64, nk, kfull + 8 * st, HSub);
      tma_load_rows<W>(sV + HB * st, &map_v, (last - e) * 64, nk, kfull + 8 * st, HSub);
    };
    if (nh > 0) {
      if (lead) {
        mbar_expect_tx(qfull, TB);
        tma_load_rows<W>(sQ, &map_q, i0, n, qfull);
      }
      for (int e = 0; e < R && e < nh; ++e) load_keys(e, e);
      mbar_wait_warp(qfull, 0, ctl, &g_attend_status, kErrWaitTma);
      uint32_t pending = 0, flip = 0, side = 0;          // warpgroups with a P~ to come, the parity of the next, the buffer of its scores
      // (counters in place of remainders: this warp's time between two products is what the others wait for)
      int in = 0, out = 0, refill = 0;
      uint32_t phase = 0, back = 0, word = 0, hole = 0;
      for (int e = 0; e < nh + 2; ++e) {
        const int hh = last - e;
        if (((hh & 31) == 31 || e == 0) && e < nh) {
          const int x = (hh & ~31) + lane, what = hh < kStates || x >= h0 + nh ? 0 : state(x);
          word = uniform(hh < kStates ? s_state.any(hh) : __ballot_sync(0xffffffffu, what != 0));
          hole = uniform(hh < kStates ? s_state.holes(hh) : __ballot_sync(0xffffffffu, what == 3));
        }
        if (e < nh) {
          mbar_wait_warp(kfull + 8 * in, phase, ctl, &g_attend_status, kErrWaitTma);
          if (hole >> (hh & 31) & 1) {
            zero_holes<D / 64>(smem + TB + R * HB + HB * in, 0, false, r.docs + hh * 64, r.t - hh * 64);
          }
        }
        const int w = e & 1;
        const uint32_t tW = tmem + F::kWgCols * w;
        const bool seen = e < nh && (word >> (hh & 31) & 1), old = pending >> w & 1;
        const int was = side >> w & 1, now = NB == 2 ? was ^ 1 : 0;
        auto scores = [&]() {
          tc_fence_after();
          mma_scores_wide<W>(lead, tW + 64 * now, dQ, kTileBytes, Desc{dK.lo + (HB >> 4) * in, dK.hi},
                             HSub, id_s);
          mma_commit(lead, sdone + 8 * (NB * w + now));   // the scores, and every product in front of them
        };
        if (NB == 2 && seen) scores();                   // into the other buffer, while the arithmetic is at the last ones
        if (old) {                                       // of half tile e - 2
          const int bar = NB * w + (NB == 2 ? was : 0);
          mbar_wait_warp(pready + 8 * bar, flip >> bar & 1, ctl, &g_attend_status, kErrWaitTile);
          flip ^= 1u << bar;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)                 // 16 keys per instruction: 16 rows of 128 B = 128 units
            mma_ts(lead, tW + 64 * NB, tW + 64 * (NB == 2 ? was : 0) + 8 * kk, dV, (HB >> 4) * out + 128 * kk, id_p, 1);
          if (NB == 2) mma_commit(lead, odone + 8 * w);
        }
        if (NB == 1 && seen) scores();
        pending = seen ? pending | 1u << w : pending & ~(1u << w);
        if (NB == 2 && seen) side ^= 1u << w;
        if (e >= 2) {
          mma_commit(lead, kfree + 8 * out);
          if (++out == R) out = 0;
        }
        // half tile e - 3, whose products were issued one round ago, makes room for e - 3 + R
        if (e >= 3) {
          if (e - 3 + R < nh) {
            mbar_wait_warp(kfree + 8 * refill, back, ctl, &g_attend_status, kErrWaitMma);
            load_keys(e - 3 + R, refill);
          }
          if (++refill == R) { refill = 0; back ^= 1; }
        }
        if (++in == R) { in = 0; phase ^= 1; }
      }
#pragma unroll
      for (int w = 0; w < NG; ++w)
        if (NB == 1) mma_commit(lead, sdone + 8 * w);                                // the last products
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ the compute warps: lane = query
    const uint32_t tS = tmem + F::kWgCols * wg + ((uint32_t)((warp & 3) * 32) << 16), tO = tS + 64 * NB;
    {
      uint32_t z[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) z[c] = 0u;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) tmem_st16(tO + 16 * c, z);
      tmem_st_wait();
    }
    const int half = wg & 1, i = i0 + row, is = min(i, r.t - 1);
    float ref = -INFINITY, s = 0.f, sr = 0.f;
    int turn = 0;
    for (int e = half; e < nh; e += 2) {
      const int hh = last - e, what = (int)uniform(hh < kStates ? s_state.of(hh) : state(hh));
      if (what == 0) continue;
      // (two buffers: the first scores go to buffer 1)
      const int side = NB == 2 ? (turn & 1) ^ 1 : 0;
      mbar_wait_warp(sdone + 8 * (NB * wg + side), (NB == 2 ? turn >> 1 : turn) & 1, ctl, &g_attend_status, kErrWaitMma);
      tc_fence_after();
      // The products of the half tiles before this one are through.  Every turn asks before it lets its own products start, so that the
      // barrier is never more than one phase from the one asked for, where parities would be taken for one another.
      auto settled = [&]() {
        if (NB == 2 && turn > 0) {
          mbar_wait_warp(odone + 8 * wg, (turn - 1) & 1, ctl, &g_attend_status, kErrWaitMma);
          tc_fence_after();
        }
      };
      forward_step<D, CAP, BIAS>(tS + 64 * side, tO, r, lin, pre, hh * 64, is, what & 1, ref, s, sr, settled);
      settled();
      ++turn;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pready + 8 * (NB * wg + side));
    }
    if (NB == 2 ? turn > 0 : nh > 0)
      mbar_wait_warp(NB == 2 ? odone + 8 * wg : sdone + 8 * wg, (NB == 2 ? turn - 1 : turn) & 1, ctl, &g_attend_status, kErrWaitMma);
    tc_fence_after();
    // every product has read the ring, which the merge goes over
    asm volatile("bar.sync 1, %0;" ::"n"(256) : "memory");
    // Each of a tile's two warpgroups finishes half of the features: it hands the other half of its accumulator over.
    constexpr int kPart = D / 2;
    float* sX = reinterpret_cast<float*>(smem + TB);                                 // [2][128][kPart]
    float* rounded = reinterpret_cast<float*>(sStat + 256);
    sStat[half * 128 + row] = make_float2(ref, s);
    rounded[half * 128 + row] = sr;
    float* give = sX + ((1 - half) * 128 + row) * kPart;
    __syncwarp();
#pragma unroll
    for (int c0 = 0; c0 < kPart; c0 += 32) {
      float o[32];
      tmem_ld32(tO + kPart * (1 - half) + c0, o);
      tmem_ld_wait(o);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        reinterpret_cast<float4*>(give + c0)[c ^ (row & 7)] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
    }
    auto meet = [] { asm volatile("bar.sync 2, 256;" ::: "memory"); };
    meet();
    const float2 other = sStat[(1 - half) * 128 + row];
    const float m = fmaxf(ref, other.x), base = m == -INFINITY ? 0.f : m;
    const float f_own = fast_exp2(ref - base), f_oth = fast_exp2(other.x - base);
    const float den = s * f_own + other.y * f_oth, by = sr * f_own + rounded[(1 - half) * 128 + row] * f_oth, inv = by == 0.f ? 0.f : 1.f / by;
    __syncwarp();
    const float a_own = f_own * inv, a_oth = f_oth * inv;
    const float* take = sX + (half * 128 + row) * kPart;
    bool bad = false;
#pragma unroll
    for (int c0 = 0; c0 < kPart; c0 += 32) {
      float o[32];
      __syncwarp();
      tmem_ld32(tO + kPart * half + c0, o);
      tmem_ld_wait(o);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 x = reinterpret_cast<const float4*>(take + c0)[c ^ (row & 7)];
        o[4 * c] = o[4 * c] * a_own + x.x * a_oth;
        o[4 * c + 1] = o[4 * c + 1] * a_own + x.y * a_oth;
        o[4 * c + 2] = o[4 * c + 2] * a_own + x.z * a_oth;
        o[4 * c + 3] = o[4 * c + 3] * a_own + x.w * a_oth;
      }
      float sum = 0.f;                                    // not finite if any of them is not
#pragma unroll
      for (int c = 0; c < 32; ++c) sum = fmaf(o[c], 0.f, sum);
      bad = bad || sum != 0.f;
      if (i < r.t) {
        const int64_t at = (((int64_t)n * a.t + i) * D + kPart * half + c0) / 8;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          reinterpret_cast<uint4*>(a.out)[at + c] =
              make_uint4(pack_pair(o[8 * c], o[8 * c + 1]), pack_pair(o[8 * c + 2], o[8 * c + 3]),
                         pack_pair(o[8 * c + 4], o[8 * c + 5]), pack_pair(o[8 * c + 6], o[8 * c + 7]));
        if (a.rest != nullptr) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            reinterpret_cast<uint4*>(a.rest)[at + c] =
                make_uint4(left_pair(o[8 * c], o[8 * c + 1]), left_pair(o[8 * c + 2], o[8 * c + 3]),
                           left_pair(o[8 * c + 4], o[8 * c + 5]), left_pair(o[8 * c + 6], o[8 * c + 7]));
        }
      }
    }
    if (half == 0 && i < r.t && a.lse != nullptr) a.lse[(int64_t)n * a.t + i] = den == 0.f ? INFINITY : m + log2f(den);
    if (bad && i < r.t) sFlag[row] = 1;
    meet();
    // (both warpgroups have written their halves; a warp's rows are its own lanes', every other one of them)
    unsigned again = __ballot_sync(0xffffffffu, sFlag[row] != 0) & (half ? 0xaaaaaaaau : 0x55555555u);
    if (again) attend::redo_rows<attend::kRedoForward, __nv_bfloat16, D>(a, b, h, i0 + (row & 96), again);
  }
  drain_if_aborted(ctl);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free(tmem, F::kTmem);
}

// ---- backward ------------------------------------------------------------------------------------------
// STAY 0: queries stay (dq), 1: keys stay (dk, dv).  Staying tile: [Q, dout] or [K, V], rows of 128; passing half tiles: [K, V] or
// [Q, dout], rows of 64, with the passing queries' (lse, delta).
template <int D, int STAY, int NW> struct AttendBackward {
  static constexpr int kThreads = 128 * NW + 64;
  static constexpr int kRing = D == 64 ? (NW == 1 ? 4 : 6) : STAY == 1 ? 4 : 5;         // one more than are in work, at least
  static constexpr uint32_t kTile = Rows<kForm<D>>::kBytes, kHalf = kTile / 2;
  static constexpr int kAcc = STAY == 1 ? 2 * D : D;                     // accumulator columns
  static constexpr bool kHoles = D == 128 || NW == 1;                    // (heads of 64 with documents, and so with padding, take NW = 1)
  static_assert(NW * 128 + kAcc <= 512, "the warpgroups' scores and the accumulators fit TMEM");
  static constexpr int kTmem = NW * 128 + kAcc <= 256 ? 256 : 512, kPerSm = D == 64 && kTmem == 256 ? 2 : 1;
  // staying tiles | passing tiles [ring] x 2 | (lse, delta) [ring][64] | flags [128] | barriers + control
  static constexpr int kOperands = (int)(2 * kTile + 2 * kRing * kHalf);
  static constexpr int kStats = STAY == 1 ? kRing * 512 : 0;
  static constexpr int kBytes = kOperands + kStats + 512 + 256 + 1024;
  static_assert(kBytes + (int)sizeof(States) + 256 <= 232448, "shared memory, with what the kernel has of its own");
};

// Bytes of global memory into shared memory, both on 16-byte boundaries.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}

// A warpgroup's step over 64 columns: S at tS, dout . v at tS + 64.  P (keys stay) as bf16 over the scores and dS over the
// others, both as A operands.  x0: the first passing token, y: the lane's own; st: (-lse, -lse, -delta, -delta) of pairs of passing
// queries; own: (-lse, -delta) of the lane's query.  EDGE: bits say which of the passing tokens count.
template <int STAY, bool CAP, bool BIAS, bool EDGE>
__device__ __forceinline__ void backward_tile(uint32_t tS, const Row& r, float lin, float pre, int x0, int y, float2 own, const float4* st,
                                              const uint2& bits) {
#pragma unroll
  for (int c0 = 0; c0 < 64; c0 += 32) {
    float v[32], g[32];
    tmem_ld32(tS + c0, v);
    tmem_ld32(tS + 64 + c0, g);
    tmem_ld_wait(v);
    tmem_ld_wait(g);
    if (CAP) cap_scores<32>(v, pre, r.cap2 > kWideCap * kLog2e);
    uint32_t pw[16], gw[16];
    const float2 mm = make_float2(lin, lin);
    // the distance's term of column e: first + step * e; in masked tiles, whose distances have both signs, these are the plain
    // distances, and the slope, of either sign itself, comes to their size
    const float by = EDGE ? 1.f : r.slope2, step = STAY == 1 ? -by : by;
    const float first = by * (float)(STAY == 1 ? y - x0 - c0 : x0 + c0 - y);
    const float2 slope = make_float2(-r.slope2, -r.slope2);
    float2 far = make_float2(first, first + step);
    const float2 two = make_float2(2.f * step, 2.f * step);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float2 off = make_float2(own.x, own.x), delta = make_float2(own.y, own.y);
      if (STAY == 1) {
        const float4 x = st[(c0 + e) >> 1];
        off = make_float2(x.x, x.y);
        delta = make_float2(x.z, x.w);
      }
      if (BIAS) {
        off = EDGE ? fma2(make_float2(fabsf(far.x), fabsf(far.y)), slope, off) : add2(off, far);
        far = add2(far, two);
      }
      const float2 z = fma2(make_float2(v[e], v[e + 1]), mm, off);
      float2 p = make_float2(fast_exp2(z.x), fast_exp2(z.y));
      float2 d = mul2(p, add2(make_float2(g[e], g[e + 1]), delta));
      if (CAP) {
        const float2 t = make_float2(v[e], v[e + 1]);
        d = sub2(d, mul2(mul2(t, t), d));
      }
      if (EDGE) {
        if (!bit_of(bits, c0 + e)) p.x = d.x = 0.f;
        if (!bit_of(bits, c0 + e + 1)) p.y = d.y = 0.f;
      }
      if (STAY == 1) pw[e >> 1] = pack_pair(p.x, p.y);
      gw[e >> 1] = pack_pair(d.x, d.y);
    }
    if (STAY == 1) tmem_st16(tS + c0 / 2, pw);
    tmem_st16(tS + 64 + c0 / 2, gw);
  }
  tmem_st_wait();
}

// grid = rows * ceil(t / 128): dq: batch * heads rows, last queries first; dk, dv: batch * kv_heads rows, first keys first.
// map_a, map_b: Q and dout (batch * heads rows); map_c, map_d: K and V (batch * kv_heads rows), boxes of 64 rows all.
// stats: (-lse, -lse, -delta, -delta) of every pair of queries, padded to whole half tiles with -inf and 0.
template <int D, int STAY, int NW, bool CAP, bool BIAS>
__global__ void __launch_bounds__(AttendBackward<D, STAY, NW>::kThreads, AttendBackward<D, STAY, NW>::kPerSm) attend_backward_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ attend::Args a, const float2* __restrict__ stats) {
  using F = AttendBackward<D, STAY, NW>;
  constexpr int W = kForm<D>, R = F::kRing;
  constexpr uint32_t TB = F::kTile, HB = F::kHalf, HSub = kTileBytes / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  const uint32_t sA = smem_u32(smem), sB = sA + 2 * TB, sC = sB + R * HB, sStat = sC + R * HB;
  const float4* stat = reinterpret_cast<const float4*>(smem + F::kOperands);
  int* sFlag = reinterpret_cast<int*>(smem + F::kOperands + F::kStats);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::kOperands + F::kStats + 512);
  const uint32_t afull = smem_u32(bars), bfull = afull + 8, bfree = bfull + 8 * R, sdone = bfree + 8 * R, alldone = sdone + 8 * NW,
                 pready = alldone + 8;
  Ctl* ctl = reinterpret_cast<Ctl*>(bars + 2 + 2 * R + 2 * NW);
  __shared__ int2 s_range[F::kThreads / 32];
  __shared__ States s_state;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = tid >> 7, row = tid & 127;
  const int warp_u = uniform_warp();
  const uint32_t lead = elect_one();
  const int group = a.heads / a.kv_heads, rows = a.batch * (STAY == 1 ? a.kv_heads : a.heads);
  const int tiles = (a.t + kTileRows - 1) / kTileRows, padded = (a.t + 63) / 64 * 64;
  const int n = (int)(blockIdx.x % rows), block = (int)(blockIdx.x / rows);
  const int y0 = (STAY == 1 ? block : tiles - 1 - block) * kTileRows, y1 = min(y0 + kTileRows, a.t) - 1;
  const int b = n / (STAY == 1 ? a.kv_heads : a.heads), head = n % (STAY == 1 ? a.kv_heads : a.heads);
  const int passes = STAY == 1 ? group : 1;                      // heads whose queries pass
  Row r = attend::make_row(a, b, STAY == 1 ? head * group : head);
  const float lin = CAP ? r.cap2 : r.pre, pre = CAP ? a.scale / a.cap : 0.f;
  const Docs dy = r.ranges != nullptr ? docs_of(r, y0, y1) : Docs{INT_MAX, -1, -1, false};
  auto state = [&](int hh) {                                     // of the tile and passing half tile hh
    const int x0 = hh * 64;
    const Docs dx = r.ranges != nullptr ? docs_of(r, x0, x0 + 63) : Docs{INT_MAX, -1, -1, false};
    const int what = STAY == 1 ? pair_state<BIAS>(r, x0, x0 + 63, dx, y0, y1, dy) : pair_state<BIAS>(r, y0, y1, dy, x0, x0 + 63, dx);
    return F::kHoles && what == 1 && dx.holes ? 3 : what;
  };

  const int base = STAY == 1 ? attend::first_query(r, y0) / 64 : 0;
  const int end = STAY == 1 ? padded / 64 : (attend::key_end(r, y1) + 63) / 64;
  const int nx = STAY == 1 ? b * a.heads + head * group : b * a.kv_heads + head / group;      // the passing rows, the first of them
  auto load_passing = [&](int hh, int m, int st) {
    mbar_expect_tx(bfull + 8 * st, 2 * HB + (STAY == 1 ? 512 : 0));
    tma_load_rows<W>(sB + HB * st, STAY == 1 ? &map_q : &map_k, hh * 64, m, bfull + 8 * st, HSub);
    tma_load_rows<W>(sC + HB * st, STAY == 1 ? &map_do : &map_v, hh * 64, m, bfull + 8 * st, HSub);
    if (STAY == 1) bulk_load(sStat + 512 * st, stats + (int64_t)m * padded + hh * 64, 512, bfull + 8 * st);
  };
  // The staying tile, and for keys the queries on the diagonal, are asked for before it is known which others there are.
  const int ahead = STAY == 1 && y0 >= r.prefix ? min(2, end - base) : 0;
  if (warp_u == 4 * NW + 1 && lead) {
    ctl->abort = 0;
    for (int x = 0; x < 2 + 2 * R + NW; ++x) mbar_init(afull + 8 * x, 1);        // afull, bfull, bfree, sdone, alldone
    for (int x = 0; x < NW; ++x) mbar_init(pready + 8 * x, 4);
    fence_barrier_init();
    fence_async_smem();
    mbar_expect_tx(afull, 2 * TB);
    // (two boxes of 64 rows for each sub-tile: a box behind the last row reads zeros)
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        tma_load_rows<W>(sA + TB * x + HSub * half, STAY == 1 ? (x ? &map_v : &map_k) : (x ? &map_do : &map_q), y0 + 64 * half, n, afull,
                         kTileBytes);
    for (int e = 0; e < ahead; ++e) load_passing(base + e, nx, e);
  }
  if (tid < 128) sFlag[tid] = 0;
  __syncwarp();
  if (warp == 0) tmem_alloc(smem_u32(&ctl->tmem), F::kTmem);
  const int2 mine = keep_states(&s_state, base, end, warp, F::kThreads / 32, state);
  if (lane == 0) s_range[warp] = mine;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl->tmem), tAcc = tmem + 128 * NW;
  // passing half tiles [h0, h0 + nh) of which any sees the tile (or is seen by it), and those that are on their way
  const int2 range = all_of(s_range, F::kThreads / 32);
  const int h0 = range.y > 0 && ahead == 0 ? range.x : base, nh = range.y > 0 ? max(range.y, base + ahead) - h0 : 0, ne = nh * passes;

  if (warp_u == 4 * NW) {
    // ------------------------------------------------------------ the warp that issues MMAs
    constexpr uint32_t id_s = instr_desc(128, 64, 0, 0), id_a = instr_desc(128, D, 0, 1);
    const Desc dA = make_desc(sA, 16, 1024), dB = make_desc(sB, 16, 1024), dC = make_desc(sC, 16, 1024);
    const Desc dBm = make_desc(sB, HSub, 1024), dCm = make_desc(sC, HSub, 1024);
    if (ne > 0) {
      mbar_wait_warp(afull, 0, ctl, &g_attend_status, kErrWaitTma);
      uint32_t pending = 0, flip = 0, started = 0;         // warpgroups with a dS to come, the parity of the next
      // (counters in place of remainders: this warp's time between two products is what the others wait for)
      int w = 0, in = 0, out = 0, eh = 0;
      uint32_t phase = 0, word = 0, hole = 0;
      for (int e = 0; e < ne + NW; ++e) {
        const uint32_t tS = tmem + 128 * w;
        const int at = h0 - base + eh;
        if ((at & 31) == 0 || eh == 0) {
          const int x = (at & ~31) + lane, what = at < kStates || x >= h0 - base + nh ? 0 : state(base + x);
          word = uniform(at < kStates ? s_state.any(at) : __ballot_sync(0xffffffffu, what != 0));
          if (F::kHoles) hole = uniform(at < kStates ? s_state.holes(at) : __ballot_sync(0xffffffffu, what == 3));
        }
        if (pending >> w & 1) {                            // of half tile e - NW
          mbar_wait_warp(pready + 8 * w, flip >> w & 1, ctl, &g_attend_status, kErrWaitTile);
          flip ^= 1u << w;
          pending &= ~(1u << w);
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)                   // dS times the passing queries (or keys)
            mma_ts(lead, tAcc, tS + 64 + 8 * kk, dBm, (HB >> 4) * out + 128 * kk, id_a, started | (kk > 0));
          if (STAY == 1) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)                 // P times their dout
              mma_ts(lead, tAcc + D, tS + 8 * kk, dCm, (HB >> 4) * out + 128 * kk, id_a, started | (kk > 0));
          }
          started = 1;
        }
        if (e >= NW) {
          mma_commit(lead, bfree + 8 * out);
          if (++out == R) out = 0;
        }
        if (e < ne) {
          mbar_wait_warp(bfull + 8 * in, phase, ctl, &g_attend_status, kErrWaitTma);
          if (word >> (at & 31) & 1) {
            if (F::kHoles && hole >> (at & 31) & 1) {
              zero_holes<D / 64>(smem + 2 * TB + HB * in, R * HB, STAY == 1, r.docs + (base + at) * 64, r.t - (base + at) * 64);
            }
            tc_fence_after();
            mma_scores_wide<W>(lead, tS, dA, kTileBytes, Desc{dB.lo + (HB >> 4) * in, dB.hi}, HSub, id_s);
            mma_scores_wide<W>(lead, tS + 64, Desc{dA.lo + (TB >> 4), dA.hi}, kTileBytes, Desc{dC.lo + (HB >> 4) * in, dC.hi}, HSub,
                               id_s);
            mma_commit(lead, sdone + 8 * w);
            pending |= 1u << w;
          }
        }
        if (++w == NW) w = 0;
        if (++in == R) { in = 0; phase ^= 1; }
        if (++eh == nh) eh = 0;
      }
      mma_commit(lead, alldone);
    }
    __syncwarp();
  } else if (warp_u == 4 * NW + 1) {
    // ------------------------------------------------------------ the warp that issues copies
    if (ne == 0) {
      mbar_wait_warp(afull, 0, ctl, &g_attend_status, kErrWaitTma);
      for (int e = 0; e < ahead; ++e) mbar_wait_warp(bfull + 8 * e, 0, ctl, &g_attend_status, kErrWaitTma);
    }
    int st = 0, hh = h0, m = nx;
    uint32_t phase = 1;
    for (int e = 0; e < ne; ++e) {
      if (e >= R) mbar_wait_warp(bfree + 8 * st, phase, ctl, &g_attend_status, kErrWaitMma);
      if (e >= ahead && lead) load_passing(hh, m, st);
      __syncwarp();
      if (++st == R) { st = 0; phase ^= 1; }
      if (++hh == h0 + nh) { hh = h0; ++m; }
    }
  } else {
    // ------------------------------------------------------------ the compute warps: lane = the staying query or key
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tS = tmem + 128 * wg + lanes;
    const int y = y0 + row, ys = min(y, a.t - 1);
    float2 own = make_float2(0.f, 0.f);
    if (STAY == 0) {
      const float* pair = reinterpret_cast<const float*>(stats + ((int64_t)n * padded + (y & ~1))) + (y & 1);
      own = y < a.t ? make_float2(pair[0], pair[2]) : make_float2(-INFINITY, 0.f);
    }
    int turn = 0, pass = 0, eh = wg;
    for (int e = wg; e < ne; e += NW, eh += NW) {
      while (eh >= nh) { eh -= nh; ++pass; }
      if (STAY == 1 && BIAS) r.slope2 = a.slopes[head * group + pass] * kLog2e;
      const int hh = h0 + eh, what = (int)uniform(hh - base < kStates ? s_state.of(hh - base) : state(hh));
      if (what == 0) continue;
      // which pairs count is asked for while the scores are under way; of a masked half tile most warps have all pairs or none
      uint2 bits = make_uint2(~0u, ~0u);
      bool edge = what & 1, none = false;
      if (edge) {
        bits = STAY == 1 ? query_bits(r, hh * 64, ys) : key_bits(r, ys, hh * 64);
        none = __all_sync(0xffffffffu, (bits.x | bits.y) == 0);
        edge = !__all_sync(0xffffffffu, (bits.x & bits.y) == ~0u && (!BIAS || (STAY == 1 ? ys <= hh * 64 : hh * 64 + 63 <= ys)));
      }
      mbar_wait_warp(sdone + 8 * wg, turn & 1, ctl, &g_attend_status, kErrWaitMma);
      ++turn;
      tc_fence_after();
      if (none) {
        uint32_t z[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) z[c] = 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st16(tS + (c >> 1) * 64 + (c & 1) * 16, z);
        tmem_st_wait();
      } else if (edge) {
        backward_tile<STAY, CAP, BIAS, true>(tS, r, lin, pre, hh * 64, ys, own, stat + 32 * (e % R), bits);
      } else {
        backward_tile<STAY, CAP, BIAS, false>(tS, r, lin, pre, hh * 64, ys, own, stat + 32 * (e % R), bits);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pready + 8 * wg);
    }
    if (ne > 0) mbar_wait_warp(alldone, 0, ctl, &g_attend_status, kErrWaitMma);
    tc_fence_after();
    bool bad = false;
    for (int c0 = 32 * wg; c0 < F::kAcc; c0 += 32 * NW) {
      float o[32];
      __syncwarp();
      tmem_ld32(tAcc + lanes + c0, o);
      tmem_ld_wait(o);
      const bool second = STAY == 1 && c0 >= D;            // dv
      const float f = second ? 1.f : a.scale;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        o[c] = ne == 0 ? 0.f : o[c] * f;
        sum = fmaf(o[c], 0.f, sum);
      }
      bad = bad || sum != 0.f;
      if (y < a.t) {
        __nv_bfloat16* base = reinterpret_cast<__nv_bfloat16*>(STAY == 0 ? a.dq : second ? a.dv : a.dk);
        uint4* dst = reinterpret_cast<uint4*>(base + ((int64_t)n * a.t + y) * D + (second ? c0 - D : c0));
#pragma unroll
        for (int c = 0; c < 4; ++c)
          dst[c] = make_uint4(pack_pair(o[8 * c], o[8 * c + 1]), pack_pair(o[8 * c + 2], o[8 * c + 3]),
                              pack_pair(o[8 * c + 4], o[8 * c + 5]), pack_pair(o[8 * c + 6], o[8 * c + 7]));
      }
    }
    if (bad && y < a.t) sFlag[row] = 1;
    asm volatile("bar.sync 1, %0;" ::"n"(128 * NW) : "memory");
    // rows that are not finite, each by one warp: rows and warps are told apart by their number modulo the warpgroups
    unsigned again = __ballot_sync(0xffffffffu, sFlag[row] != 0 && row % NW == wg);
    if (again) attend::redo_rows<STAY == 0 ? attend::kRedoDq : attend::kRedoDkv, __nv_bfloat16, D>(a, b, head, y0 + (row & 96), again);
  }
  drain_if_aborted(ctl);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free(tmem, F::kTmem);
}

// lse and delta_i of every query, padded, as the kernels above read them.  D / 8 lanes a row, 16 bytes each.
template <int D>
__global__ void __launch_bounds__(256) attend_stats_kernel(attend::Args a, float2* __restrict__ stats) {
  constexpr int L = D / 8;
  const int padded = (a.t + 63) / 64 * 64;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L, n = at / padded;
  const int i = (int)(at % padded), u = threadIdx.x % L;
  const bool real = n < (int64_t)a.batch * a.heads && i < a.t;
  float s = real ? attend::delta_part<__nv_bfloat16>(a, (n * a.t + i) * L + u) : 0.f;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (u == 0 && n < (int64_t)a.batch * a.heads) {
    float* pair = reinterpret_cast<float*>(stats + (at & ~(int64_t)1)) + (at & 1);
    pair[0] = real ? -a.lse[n * a.t + i] : -INFINITY;
    pair[2] = real ? -s : 0.f;
    if (real) a.delta[n * a.t + i] = s;
  }
}

}  // namespace tc
}  // namespace dil
