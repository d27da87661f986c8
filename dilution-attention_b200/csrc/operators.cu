// extern "C" entry points of masked softmax attention and of eviction.  Argument validation, kernel selection and launches;
// declarations in include/dilution_b200.h.

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/dilution_b200.h"
#include "abi_internal.h"
#include "attend_simt.cuh"
#include "evict_kernels.cuh"
#include "tc_attend.cuh"

namespace dil {

int operators_read_status(int* code) { return read_status_word(tc::g_attend_status, code); }

namespace {

// ---- masked softmax attention ------------------------------------------------------------------
int64_t doc_spans(int64_t t) { return (t + attend::kSpan - 1) / attend::kSpan; }

int check_attend(const char* fn, const attend::Args& a, int dtype, int d) {
  if (dtype != DILUTION_F32 && dtype != DILUTION_BF16)
    return abi_fail(DILUTION_ERR_ARG, "%s: dtype must be DILUTION_F32 or DILUTION_BF16", fn);
  if (!valid_d(d)) return abi_fail(DILUTION_ERR_UNSUPPORTED, "%s: head_dim %d not in {16, 32, 64, 128}", fn, d);
  if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.t < 1 || a.heads % a.kv_heads != 0)
    return abi_fail(DILUTION_ERR_ARG, "%s: sizes must be positive and kv_heads divide heads (batch=%d heads=%d kv_heads=%d t=%d)", fn,
                    a.batch, a.heads, a.kv_heads, a.t);
  if (a.t > (1 << 30) || (double)a.batch * a.heads * (double)doc_spans(a.t) >= 2147483648.0)
    return abi_fail(DILUTION_ERR_ARG, "%s: batch * heads * blocks exceeds the grid limit", fn);
  if (!valid_cap(a.cap) || !(a.scale > 0.f))
    return abi_fail(DILUTION_ERR_ARG, "%s: scale must be positive and cap in [1e-30, 1e38], or 0 for none", fn);
  if (!a.q || !a.k || !a.v || !a.out || (a.docs && !a.ranges)) return abi_fail(DILUTION_ERR_ARG, "%s: null pointer", fn);
  if (a.rest && dtype != DILUTION_BF16) return abi_fail(DILUTION_ERR_ARG, "%s: rest is of bf16 outputs alone", fn);
  if (misaligned({a.q, a.k, a.v, a.out, a.rest, a.dout, a.dq, a.dk, a.dv, a.ranges}))
    return abi_fail(DILUTION_ERR_ARG, "%s: tensors must be 16-byte aligned", fn);
  return DILUTION_OK;
}

int launch_ranges(const attend::Args& a, cudaStream_t st) {
  if (!a.docs) return DILUTION_OK;
  LaunchMark mark("attend_ranges", st);
  const int64_t spans = a.batch * doc_spans(a.t);
  attend::doc_ranges_kernel<<<(unsigned)((spans + 7) / 8), 256, 0, st>>>(a.docs, a.batch, a.t,
                                                                        const_cast<attend::DocRange*>(a.ranges));
  return abi_check_launch("attend_ranges");
}

// CTAs that share a block of `stream` tiles: until every SM has one, or each has two tiles.
template <typename K> int launch_shared(K kernel, const char* name, int64_t blocks, int64_t stream, int smem, const attend::Args& a,
                                        cudaStream_t st) {
  int ranks = 1;
  while (ranks < 8 && blocks * ranks < 148 && stream >= 2 * ranks) ranks *= 2;
  if (int rc = opt_in(kernel, smem)) return rc;
  LaunchMark mark(name, st);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(blocks * ranks));
  cfg.blockDim = dim3(attend::kSimtThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, ranks);
  return e == cudaSuccess ? DILUTION_OK : abi_fail(DILUTION_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

template <typename T, int D> int simt_forward(const attend::Args& a, cudaStream_t st) {
  return launch_shared(attend::simt_forward_kernel<T, D>, "attend_forward", (int64_t)a.batch * a.heads * doc_spans(a.t), doc_spans(a.t),
                       attend::simt_smem<D>(3), a, st);
}

template <typename T, int D> int launch_delta(const attend::Args& a, cudaStream_t st) {
  LaunchMark mark("attend_delta", st);
  const int64_t rows = (int64_t)a.batch * a.heads * a.t, threads = rows * D * (int)sizeof(T) / 16;
  attend::delta_kernel<T, D><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a, rows);
  return abi_check_launch("attend_delta");
}

template <typename T, int D> int simt_backward(const attend::Args& a, cudaStream_t st) {
  constexpr int smem = attend::simt_smem<D>(3);
  if (int rc = launch_delta<T, D>(a, st)) return rc;
  if (int rc = launch_shared(attend::simt_dkv_kernel<T, D>, "attend_dkv", (int64_t)a.batch * a.kv_heads * doc_spans(a.t),
                             doc_spans(a.t) * (a.heads / a.kv_heads), smem, a, st)) return rc;
  return launch_shared(attend::simt_dq_kernel<T, D>, "attend_dq", (int64_t)a.batch * a.heads * doc_spans(a.t), doc_spans(a.t), smem, a, st);
}

// ---- the same on the tensor cores
struct AttendMaps {
  CUtensorMap q, k, v, dout;
};
int attend_maps(AttendMaps& m, const attend::Args& a, int d, int q_box, int k_box) {
  const int64_t nq = (int64_t)a.batch * a.heads, nk = (int64_t)a.batch * a.kv_heads;
  if (!tc::tile_map(&m.q, a.q, nq, a.t, d, q_box) || !tc::tile_map(&m.k, a.k, nk, a.t, d, k_box) ||
      !tc::tile_map(&m.v, a.v, nk, a.t, d, k_box) || (a.dout && !tc::tile_map(&m.dout, a.dout, nq, a.t, d, q_box)))
    return abi_fail(DILUTION_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  return DILUTION_OK;
}
// f(bool_constant<cap>, bool_constant<bias>)
template <typename F> int with_score(const attend::Args& a, F f) {
  if (a.cap > 0.f) return a.slopes ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
  return a.slopes ? f(std::false_type(), std::true_type()) : f(std::false_type(), std::false_type());
}

template <int D> int tc_forward(const attend::Args& a, cudaStream_t st) {
  using F = tc::AttendForward<D>;
  AttendMaps m;
  if (int rc = attend_maps(m, a, D, 128, 64)) return rc;
  return with_score(a, [&](auto cap, auto bias) {
    auto kernel = tc::attend_forward_kernel<D, cap(), bias()>;
    if (int rc = opt_in(kernel, F::kBytes)) return rc;
    LaunchMark mark("attend_forward", st);
    const unsigned grid = (unsigned)((int64_t)a.batch * a.heads * ((a.t + 127) / 128));
    kernel<<<grid, F::kThreads, F::kBytes, st>>>(m.q, m.k, m.v, a);
    return abi_check_launch("attend_forward");
  });
}

template <int D, int STAY, int NW> int tc_backward_half(const attend::Args& a, const AttendMaps& m, const float2* stats, cudaStream_t st) {
  using F = tc::AttendBackward<D, STAY, NW>;
  return with_score(a, [&](auto cap, auto bias) {
    auto kernel = tc::attend_backward_kernel<D, STAY, NW, cap(), bias()>;
    if (int rc = opt_in(kernel, F::kBytes)) return rc;
    LaunchMark mark(STAY ? "attend_dkv" : "attend_dq", st);
    const unsigned grid = (unsigned)((int64_t)a.batch * (STAY ? a.kv_heads : a.heads) * ((a.t + 127) / 128));
    kernel<<<grid, F::kThreads, F::kBytes, st>>>(m.q, m.dout, m.k, m.v, a, stats);
    return abi_check_launch("attend_backward");
  });
}

template <int D> int tc_backward(const attend::Args& a, float2* stats, cudaStream_t st) {
  AttendMaps m;
  if (int rc = attend_maps(m, a, D, 64, 64)) return rc;
  {
    LaunchMark mark("attend_delta", st);
    const int64_t threads = (int64_t)a.batch * a.heads * ((a.t + 63) / 64 * 64) * (D / 8);
    tc::attend_stats_kernel<D><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a, stats);
    if (int rc = abi_check_launch("attend_delta")) return rc;
  }
  // Heads of 64: two CTAs with a warpgroup each on an SM, whose starts and ends overlap, or one with three.  dk, dv and dq in us,
  // two / one: n = 148, T = 512 25 + 19 / 31 + 24, T = 1024 68 + 54 / 79 + 64; n = 96, T = 2048 144 + 111 / 147 + 121; n = 64, T = 3000
  // 184 + 149 / 181 + 155, T = 4096 324 + 249 / 294 + 248, T = 8192 1206 + 910 / 1066 + 881; documents of 700 tokens, T = 4096
  // 120 + 95 / 143 + 115, T = 8192 235 + 185 / 281 + 230.
  if constexpr (D == 64) {
    if (a.docs || a.t <= 2560) {
      if (int rc = tc_backward_half<D, 1, 1>(a, m, stats, st)) return rc;
      return tc_backward_half<D, 0, 1>(a, m, stats, st);
    }
  }
  if (int rc = tc_backward_half<D, 1, D == 64 ? 3 : 2>(a, m, stats, st)) return rc;
  return tc_backward_half<D, 0, 3>(a, m, stats, st);
}

template <typename T, int D> constexpr bool kOnTensorCores = std::is_same<T, __nv_bfloat16>::value && (D == 64 || D == 128);

// delta (batch * heads, t) fp32, then (lse, delta) padded to half tiles.
size_t delta_bytes(int64_t batch, int64_t heads, int64_t t) { return (size_t)((batch * heads * t * 4 + 255) / 256 * 256); }

attend::Args attend_args(const void* q, const void* k, const void* v, int64_t batch, int64_t heads, int64_t kv_heads, int64_t t,
                         float scale, float cap, const float* slopes, const int* documents, const int* prefix, void* ranges,
                         void* out, void* rest, float* lse) {
  attend::Args a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.rest = rest;
  a.lse = lse;
  a.slopes = slopes;
  a.docs = documents;
  a.ranges = (const attend::DocRange*)ranges;
  a.prefix = prefix;
  // (sizes past the limits of check_attend are refused there: none of them may wrap into range)
  auto narrow = [](int64_t x) { return x > INT_MAX || x < 0 ? -1 : (int)x; };
  a.batch = narrow(batch);
  a.heads = narrow(heads);
  a.kv_heads = narrow(kv_heads);
  a.t = narrow(t);
  a.scale = scale;
  a.cap = cap;
  return a;
}

}  // namespace
}  // namespace dil

using namespace dil;

extern "C" {

size_t dilution_attend_ranges_bytes(int64_t batch, int64_t t) {
  return batch < 1 || t < 1 ? 0 : (size_t)(batch * doc_spans(t)) * sizeof(attend::DocRange);
}

size_t dilution_attend_scratch_bytes(int64_t batch, int64_t heads, int64_t t) {
  return batch < 1 || heads < 1 || t < 1 ? 0 : delta_bytes(batch, heads, t) + (size_t)(batch * heads * ((t + 63) / 64 * 64)) * 8;
}

int dilution_attend_forward(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t heads,
                            int64_t kv_heads, int64_t t, int d, float scale, float cap, const float* slopes,
                            const int* documents, const int* prefix, void* ranges, void* out, void* rest, float* lse,
                            void* stream) {
  const attend::Args a = attend_args(q, k, v, batch, heads, kv_heads, t, scale, cap, slopes, documents, prefix, ranges, out, rest, lse);
  if (int rc = check_attend("dilution_attend_forward", a, dtype, d)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = launch_ranges(a, st)) return rc;
  return with_type(dtype, d, [&](auto type, auto dim) {
    if constexpr (!kOnTensorCores<decltype(type), dim()>) return simt_forward<decltype(type), dim()>(a, st);
    else return tc_forward<dim()>(a, st);
  });
}

int dilution_attend_backward(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t heads,
                             int64_t kv_heads, int64_t t, int d, float scale, float cap, const float* slopes,
                             const int* documents, const int* prefix, const void* ranges, const void* out, const void* rest,
                             const float* lse, const void* dout, void* scratch, void* dq, void* dk, void* dv, void* stream) {
  attend::Args a = attend_args(q, k, v, batch, heads, kv_heads, t, scale, cap, slopes, documents, prefix,
                               const_cast<void*>(ranges), const_cast<void*>(out), const_cast<void*>(rest), const_cast<float*>(lse));
  a.dout = dout;
  a.delta = (float*)scratch;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  if (int rc = check_attend("dilution_attend_backward", a, dtype, d)) return rc;
  if (!lse || !dout || !scratch || !dq || !dk || !dv || misaligned({scratch})) return abi_fail(DILUTION_ERR_ARG, "dilution_attend_backward: null or misaligned pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    if constexpr (kOnTensorCores<decltype(type), dim()>)
      return tc_backward<dim()>(a, (float2*)((char*)scratch + delta_bytes(batch, heads, t)), st);
    else return simt_backward<decltype(type), dim()>(a, st);
  });
}

int dilution_evict(const void* k_cache, const void* v_cache, const float* committed, int dtype, int64_t n, int64_t capacity,
                   int64_t length, int d, const float* scores, int64_t score_stride, int64_t keep, int64_t recent, int64_t sinks,
                   int64_t new_capacity, void* k_out, void* v_out, float* committed_out, int* index, void* stream) {
  if (dtype != DILUTION_F32 && dtype != DILUTION_BF16)
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: dtype must be DILUTION_F32 or DILUTION_BF16");
  if (!valid_d(d)) return abi_fail(DILUTION_ERR_UNSUPPORTED, "dilution_evict: head_dim %d not in {16, 32, 64, 128}", d);
  if (n < 1 || n > (1 << 24) || capacity < 1 || capacity > (1 << 30) || length < 1 || length > capacity || score_stride < length)
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: length %lld outside cache capacity %lld", (long long)length, (long long)capacity);
  if (recent < 0 || sinks < 0 || keep < 1 || keep > length || recent > keep || sinks > keep - recent)
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: keep %lld of %lld keys with %lld recent and %lld first ones", (long long)keep,
                    (long long)length, (long long)recent, (long long)sinks);
  const int per = d * (dtype == DILUTION_F32 ? 4 : 2) / 16;
  if (new_capacity < keep || new_capacity > (1 << 25) || n * (new_capacity * per / 1024 + 1) >= (int64_t)1 << 31)
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: new capacity %lld", (long long)new_capacity);
  if (!k_cache || !v_cache || !scores || !k_out || !v_out || !index || (committed == nullptr) != (committed_out == nullptr))
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: null pointer");
  if (misaligned({k_cache, v_cache, k_out, v_out})) return abi_fail(DILUTION_ERR_ARG, "dilution_evict: caches must be 16-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  // CTAs of a row: until all SMs have one or a CTA has 256 keys, and until a CTA has 8192 keys
  int ranks = 1;
  while (ranks < 8 && n * ranks < 148 && length / (2 * ranks) >= 256) ranks *= 2;
  while (ranks < 8 && (length + ranks - 1) / ranks > 8192) ranks *= 2;
  evict::Args a{};
  a.scores = scores;
  a.score_stride = score_stride;
  a.length = (int)length;
  a.keep = (int)keep;
  a.recent = (int)recent;
  a.sinks = (int)sinks;
  a.seg = (int)((length + ranks - 1) / ranks);
  a.held = a.seg <= evict::kMaxHeld;
  a.index = index;
  a.k = (const uint4*)k_cache;
  a.v = (const uint4*)v_cache;
  a.committed = committed;
  a.capacity = capacity;
  a.new_capacity = (int)new_capacity;
  while (1 << a.shift < per) ++a.shift;
  a.moves = n * ranks >= 148;
  a.k_out = (uint4*)k_out;
  a.v_out = (uint4*)v_out;
  a.committed_out = committed_out;
  if (int rc = opt_in(evict::select_kernel, evict::kMaxHeld * 4)) return rc;
  {
    LaunchMark mark("evict_select", st);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(n * ranks));
    cfg.blockDim = dim3(evict::kThreads);
    cfg.dynamicSmemBytes = a.held ? (a.seg + 3) / 4 * 16 : 0;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, evict::select_kernel, a, ranks);
    if (e != cudaSuccess) return abi_fail(DILUTION_ERR_CUDA, "evict_select: %s", cudaGetErrorString(e));
  }
  if (a.moves) return DILUTION_OK;
  LaunchMark mark("evict_gather", st);
  const int64_t blocks = n * ((new_capacity * per + 1023) / 1024);
  evict::gather_kernel<<<(unsigned)blocks, 256, 0, st>>>(a);
  return abi_check_launch("evict_gather");
}

}  // extern "C"
