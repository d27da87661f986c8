// extern "C" entry points of the operators around the attention layers: masked softmax attention, draft trees over a cache,
// eviction.  Argument validation, kernel selection and launches; declarations in include/dilution_b200.h.

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/dilution_b200.h"
#include "abi_internal.h"
#include "attend_simt.cuh"
#include "evict_kernels.cuh"
#include "once_per_device.cuh"
#include "tc_attend.cuh"
#include "tree_simt.cuh"

namespace dil {

int operators_read_status(int* code) {
  int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return 3;
  if (cudaMemcpyFromSymbol(&v, tc::g_attend_status, sizeof(int)) != cudaSuccess) return 3;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(tc::g_attend_status, &zero, sizeof(int));
  }
  *code = v;
  return 0;
}

namespace {

bool valid_d(int d) { return d == 16 || d == 32 || d == 64 || d == 128; }
bool misaligned(std::initializer_list<const void*> ps) {
  uintptr_t x = 0;
  for (const void* p : ps) x |= (uintptr_t)p;
  return x & 15;
}

template <typename K> int opt_in(K kernel, int bytes) {
  static OncePerDevice done;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  if (bytes <= 48 * 1024 || done.done((const void*)kernel, dev)) return DILUTION_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return abi_fail(DILUTION_ERR_CUDA, "cudaFuncSetAttribute(%d): %s", bytes, cudaGetErrorString(e));
  done.set((const void*)kernel, dev);
  return DILUTION_OK;
}

// f(T(), integral_constant<int, D>()) for the element type and head size.
template <typename T, typename F> int with_d(int d, F f) {
  switch (d) {
    case 16: return f(T(), std::integral_constant<int, 16>());
    case 32: return f(T(), std::integral_constant<int, 32>());
    case 64: return f(T(), std::integral_constant<int, 64>());
    default: return f(T(), std::integral_constant<int, 128>());
  }
}
template <typename F> int with_type(int dtype, int d, F f) {
  return dtype == DILUTION_F32 ? with_d<float>(d, f) : with_d<__nv_bfloat16>(d, f);
}

// ---- masked softmax attention ------------------------------------------------------------------
int64_t doc_spans(int64_t t) { return (t + attend::kSpan - 1) / attend::kSpan; }

int check_attend(const char* fn, const attend::Args& a, int dtype, int d) {
  if (dtype != DILUTION_F32 && dtype != DILUTION_BF16)
    return abi_fail(DILUTION_ERR_ARG, "%s: dtype must be DILUTION_F32 or DILUTION_BF16", fn);
  if (!valid_d(d)) return abi_fail(DILUTION_ERR_UNSUPPORTED, "%s: head_dim %d not in {16, 32, 64, 128}", fn, d);
  if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.t < 1 || a.heads % a.kv_heads != 0)
    return abi_fail(DILUTION_ERR_ARG, "%s: sizes must be positive and kv_heads divide heads (batch=%d heads=%d kv_heads=%d t=%d)", fn,
                    a.batch, a.heads, a.kv_heads, a.t);
  if (a.t > (1 << 30) || (int64_t)a.batch * a.heads * doc_spans(a.t) >= (int64_t)1 << 31)
    return abi_fail(DILUTION_ERR_ARG, "%s: batch * heads * blocks exceeds the grid limit", fn);
  if (!(a.cap >= 0.f) || a.cap > 3e38f || !(a.scale > 0.f))
    return abi_fail(DILUTION_ERR_ARG, "%s: scale must be positive and cap finite, 0 for none", fn);
  if (!a.q || !a.k || !a.v || !a.out || (a.docs && !a.ranges)) return abi_fail(DILUTION_ERR_ARG, "%s: null pointer", fn);
  if (misaligned({a.q, a.k, a.v, a.out, a.dout, a.dq, a.dk, a.dv, a.ranges}))
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

template <typename T, int D> int simt_forward(const attend::Args& a, cudaStream_t st) {
  constexpr int smem = attend::simt_smem<D>(3);
  if (int rc = opt_in(attend::simt_forward_kernel<T, D>, smem)) return rc;
  LaunchMark mark("attend_forward", st);
  const unsigned grid = (unsigned)((int64_t)a.batch * a.heads * doc_spans(a.t));
  attend::simt_forward_kernel<T, D><<<grid, attend::kSimtThreads, smem, st>>>(a);
  return abi_check_launch("attend_forward");
}

template <typename T, int D> int launch_delta(const attend::Args& a, cudaStream_t st) {
  LaunchMark mark("attend_delta", st);
  const int64_t rows = (int64_t)a.batch * a.heads * a.t, threads = rows * D * (int)sizeof(T) / 16;
  attend::delta_kernel<T, D><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>((const T*)a.dout, (const T*)a.out, rows, a.delta);
  return abi_check_launch("attend_delta");
}

template <typename T, int D> int simt_backward(const attend::Args& a, cudaStream_t st) {
  constexpr int smem = attend::simt_smem<D>(3);
  if (int rc = launch_delta<T, D>(a, st)) return rc;
  if (int rc = opt_in(attend::simt_dq_kernel<T, D>, smem)) return rc;
  if (int rc = opt_in(attend::simt_dkv_kernel<T, D>, smem)) return rc;
  {
    LaunchMark mark("attend_dkv", st);
    const unsigned grid = (unsigned)((int64_t)a.batch * a.kv_heads * doc_spans(a.t));
    attend::simt_dkv_kernel<T, D><<<grid, attend::kSimtThreads, smem, st>>>(a);
    if (int rc = abi_check_launch("attend_dkv")) return rc;
  }
  LaunchMark mark("attend_dq", st);
  const unsigned grid = (unsigned)((int64_t)a.batch * a.heads * doc_spans(a.t));
  attend::simt_dq_kernel<T, D><<<grid, attend::kSimtThreads, smem, st>>>(a);
  return abi_check_launch("attend_dq");
}

// ---- the same on the tensor cores
struct AttendMaps {
  CUtensorMap q, k, v, dout;
};
int attend_maps(AttendMaps& m, const attend::Args& a, int d, int q_box, int k_box) {
  const int64_t nq = (int64_t)a.batch * a.heads, nk = (int64_t)a.batch * a.kv_heads;
  if (!tc::attend_map(&m.q, a.q, nq, a.t, d, q_box) || !tc::attend_map(&m.k, a.k, nk, a.t, d, k_box) ||
      !tc::attend_map(&m.v, a.v, nk, a.t, d, k_box) || (a.dout && !tc::attend_map(&m.dout, a.dout, nq, a.t, d, q_box)))
    return abi_fail(DILUTION_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  return DILUTION_OK;
}
// f(bool_constant<cap>, bool_constant<bias>)
template <typename F> int with_score(const attend::Args& a, F f) {
  if (a.cap > 0.f) return a.slopes ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
  return a.slopes ? f(std::false_type(), std::true_type()) : f(std::false_type(), std::false_type());
}

template <int D, int NT> int tc_forward(const attend::Args& a, cudaStream_t st) {
  using F = tc::AttendForward<D, NT>;
  AttendMaps m;
  if (int rc = attend_maps(m, a, D, 128, 64)) return rc;
  return with_score(a, [&](auto cap, auto bias) {
    auto kernel = tc::attend_forward_kernel<D, NT, cap(), bias()>;
    if (int rc = opt_in(kernel, F::kBytes)) return rc;
    LaunchMark mark("attend_forward", st);
    const unsigned grid = (unsigned)((int64_t)a.batch * a.heads * ((a.t + 128 * NT - 1) / (128 * NT)));
    kernel<<<grid, F::kThreads, F::kBytes, st>>>(m.q, m.k, m.v, a);
    return abi_check_launch("attend_forward");
  });
}

template <int D, int STAY> int tc_backward_half(const attend::Args& a, const AttendMaps& m, const float2* stats, cudaStream_t st) {
  using F = tc::AttendBackward<D, STAY>;
  return with_score(a, [&](auto cap, auto bias) {
    auto kernel = tc::attend_backward_kernel<D, STAY, cap(), bias()>;
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
  if (int rc = tc_backward_half<D, 1>(a, m, stats, st)) return rc;
  return tc_backward_half<D, 0>(a, m, stats, st);
}

bool on_tensor_cores(int dtype, int d) { return dtype == DILUTION_BF16 && (d == 64 || d == 128); }

// delta (batch * heads, t) fp32, then (lse, delta) padded to half tiles.
size_t delta_bytes(int64_t batch, int64_t heads, int64_t t) { return (size_t)((batch * heads * t * 4 + 255) / 256 * 256); }

attend::Args attend_args(const void* q, const void* k, const void* v, int64_t batch, int64_t heads, int64_t kv_heads, int64_t t,
                         float scale, float cap, const float* slopes, const int* documents, const int* prefix, void* ranges,
                         void* out, float* lse) {
  attend::Args a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
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

// ---- draft trees -----------------------------------------------------------------------------------
// Parts that a key head's keys are cut into: enough blocks for four on every SM, of 256 keys at least.
int tree_chunks(int64_t blocks, int64_t keys) {
  const int64_t want = (148 * 4 + blocks - 1) / std::max<int64_t>(blocks, 1), most = (keys + 255) / 256;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, 512}));
}
int tree_row_blocks(int rows) { return rows <= 16 ? 1 : (rows + 63) / 64; }

struct TreeScratch {
  size_t part, psum, pout, bytes;
};
TreeScratch tree_scratch(int64_t heads, int64_t rows, int64_t chunks, int d) {
  TreeScratch s;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t n = (size_t)(heads * rows * chunks);
  s.part = 0;
  s.psum = up(n * sizeof(float2));
  s.pout = s.psum + up(n * sizeof(float));
  s.bytes = s.pout + n * d * sizeof(float);
  return s;
}
int64_t tree_keys(const tree::Args& a) { return (a.pos_dev ? a.capacity : a.len) + a.nodes; }

int check_tree(const char* fn, const tree::Args& a, int64_t length, int dtype, int d) {
  if (dtype != DILUTION_F32 && dtype != DILUTION_BF16)
    return abi_fail(DILUTION_ERR_ARG, "%s: dtype must be DILUTION_F32 or DILUTION_BF16", fn);
  if (!valid_d(d)) return abi_fail(DILUTION_ERR_UNSUPPORTED, "%s: head_dim %d not in {16, 32, 64, 128}", fn, d);
  if (a.batch < 1 || a.kv_heads < 1 || a.group < 1 || (int64_t)a.batch * a.kv_heads > 65535 || a.group > 1024)
    return abi_fail(DILUTION_ERR_ARG, "%s: batch * kv_heads must be in [1, 65535] and the heads of a group in [1, 1024]", fn);
  if (a.nodes < 1 || a.nodes > tree::kMaxNodes)
    return abi_fail(DILUTION_ERR_ARG, "%s: a tree has 1 to %d nodes, not %d", fn, tree::kMaxNodes, a.nodes);
  if (a.capacity < 1 || a.capacity > (1 << 30) || length < 0 || length > a.capacity)
    return abi_fail(DILUTION_ERR_ARG, "%s: length %lld outside cache capacity %lld", fn, (long long)length, (long long)a.capacity);
  if (!(a.cap >= 0.f) || a.cap > 3e38f || !(a.scale > 0.f))
    return abi_fail(DILUTION_ERR_ARG, "%s: scale must be positive and cap finite, 0 for none", fn);
  if (!a.q || !a.kn || !a.vn || !a.kc || !a.vc || !a.parents || !a.lse) return abi_fail(DILUTION_ERR_ARG, "%s: null pointer", fn);
  if (misaligned({a.q, a.kn, a.vn, a.kc, a.vc}))
    return abi_fail(DILUTION_ERR_ARG, "%s: q, drafted keys and values and caches must be 16-byte aligned", fn);
  return DILUTION_OK;
}

tree::Args tree_args(const void* q, const void* k_new, const void* v_new, const void* k_cache, const void* v_cache,
                     const int* parents, int64_t parent_stride, int64_t batch, int64_t kv_heads, int group, int nodes,
                     int64_t capacity, int64_t length, const int* length_dev, float scale, float* lse) {
  tree::Args a{};
  a.q = q;
  a.kn = k_new;
  a.vn = v_new;
  a.kc = k_cache;
  a.vc = v_cache;
  a.parents = parents;
  a.parent_stride = parent_stride;
  a.pos_dev = length_dev;
  a.lse = lse;
  a.capacity = capacity;
  a.len = (int)std::min<int64_t>(length, INT_MAX);
  a.batch = batch > INT_MAX || batch < 0 ? -1 : (int)batch;
  a.kv_heads = kv_heads > INT_MAX || kv_heads < 0 ? -1 : (int)kv_heads;
  a.group = group;
  a.nodes = nodes;
  a.scale = scale;
  return a;
}

void place_scratch(tree::Args& a, void* scratch, int rows, int d) {
  const TreeScratch s = tree_scratch((int64_t)a.batch * a.kv_heads, rows, a.chunks, d);
  char* p = (char*)scratch;
  a.part = (float2*)(p + s.part);
  a.psum = (float*)(p + s.psum);
  a.pout = (float*)(p + s.pout);
}

template <typename T, int D, int RI, bool OUT> int simt_softmax(const tree::Args& a, cudaStream_t st) {
  constexpr int smem = sizeof(tree::Smem<D, RI>);
  if (int rc = opt_in(tree::simt_softmax_kernel<T, D, RI, OUT>, smem)) return rc;
  LaunchMark mark(OUT ? "tree_softmax" : "tree_stats", st);
  const dim3 grid(a.chunks, (a.group * a.nodes + 16 * RI - 1) / (16 * RI), a.batch * a.kv_heads);
  tree::simt_softmax_kernel<T, D, RI, OUT><<<grid, tree::kThreads, smem, st>>>(a);
  return abi_check_launch("tree_softmax");
}
template <typename T, int D, int RI> int simt_dilute(const tree::Args& a, cudaStream_t st) {
  constexpr int smem = sizeof(tree::Smem<D, RI>);
  if (int rc = opt_in(tree::simt_dilute_kernel<T, D, RI>, smem)) return rc;
  LaunchMark mark("tree_dilute", st);
  tree::simt_dilute_kernel<T, D, RI><<<dim3(a.chunks, 1, a.batch * a.kv_heads), tree::kThreads, smem, st>>>(a);
  return abi_check_launch("tree_dilute");
}
template <typename T, int D, int RI> int simt_advance(const tree::Args& a, const tree::Accept& c, cudaStream_t st) {
  constexpr int smem = sizeof(tree::Smem<D, RI>);
  if (int rc = opt_in(tree::simt_advance_kernel<T, D, RI>, smem)) return rc;
  LaunchMark mark("tree_advance", st);
  const int64_t tiles = ((a.pos_dev ? a.capacity : a.len) + c.accepted + tree::kKeys - 1) / tree::kKeys;
  tree::simt_advance_kernel<T, D, RI>
      <<<dim3((unsigned)std::min<int64_t>(tiles, a.chunks), 1, a.batch * a.kv_heads), tree::kThreads, smem, st>>>(a, c);
  return abi_check_launch("tree_advance");
}

template <typename T, bool DILUTE> int join(const tree::Args& a, int d, cudaStream_t st) {
  LaunchMark mark("tree_join", st);
  tree::join_kernel<T, DILUTE><<<(unsigned)((int64_t)a.batch * a.kv_heads * a.group * a.nodes), d, 0, st>>>(a, d);
  return abi_check_launch("tree_join");
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
                            const int* documents, const int* prefix, void* ranges, void* out, float* lse, void* stream) {
  const attend::Args a = attend_args(q, k, v, batch, heads, kv_heads, t, scale, cap, slopes, documents, prefix, ranges, out, lse);
  if (int rc = check_attend("dilution_attend_forward", a, dtype, d)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = launch_ranges(a, st)) return rc;
  if (on_tensor_cores(dtype, d)) {
    if (d == 128) return tc_forward<128, 1>(a, st);
    return (int64_t)a.batch * a.heads * ((a.t + 255) / 256) >= 148 ? tc_forward<64, 2>(a, st) : tc_forward<64, 1>(a, st);
  }
  return with_type(dtype, d, [&](auto type, auto dim) { return simt_forward<decltype(type), dim()>(a, st); });
}

int dilution_attend_backward(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t heads,
                             int64_t kv_heads, int64_t t, int d, float scale, float cap, const float* slopes,
                             const int* documents, const int* prefix, const void* ranges, const void* out, const float* lse,
                             const void* dout, void* scratch, void* dq, void* dk, void* dv, void* stream) {
  attend::Args a = attend_args(q, k, v, batch, heads, kv_heads, t, scale, cap, slopes, documents, prefix,
                               const_cast<void*>(ranges), const_cast<void*>(out), const_cast<float*>(lse));
  a.dout = dout;
  a.delta = (float*)scratch;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  if (int rc = check_attend("dilution_attend_backward", a, dtype, d)) return rc;
  if (!lse || !dout || !scratch || !dq || !dk || !dv || misaligned({scratch})) return abi_fail(DILUTION_ERR_ARG, "dilution_attend_backward: null or misaligned pointer");
  cudaStream_t st = (cudaStream_t)stream;
  if (on_tensor_cores(dtype, d)) {
    float2* stats = (float2*)((char*)scratch + delta_bytes(batch, heads, t));
    return d == 128 ? tc_backward<128>(a, stats, st) : tc_backward<64>(a, stats, st);
  }
  return with_type(dtype, d, [&](auto type, auto dim) { return simt_backward<decltype(type), dim()>(a, st); });
}

size_t dilution_tree_scratch_bytes(int64_t batch, int64_t kv_heads, int group, int nodes, int64_t length, int d) {
  if (batch < 1 || kv_heads < 1 || group < 1 || nodes < 1 || length < 0 || d < 1) return 0;
  const int rows = group * nodes;
  return tree_scratch(batch * kv_heads, rows, tree_chunks(batch * kv_heads * tree_row_blocks(rows), length + nodes), d).bytes;
}

int dilution_tree_softmax(const void* q, const void* k_new, const void* v_new, const void* k_cache, const void* v_cache, int dtype,
                          int64_t batch, int64_t kv_heads, int group, int nodes, int64_t capacity, int64_t length,
                          const int* length_dev, int d, float scale, float cap, const float* slopes, const int* parents,
                          int64_t parent_stride, float* lse, void* out, void* scratch, void* stream) {
  tree::Args a = tree_args(q, k_new, v_new, k_cache, v_cache, parents, parent_stride, batch, kv_heads, group, nodes, capacity,
                           length, length_dev, scale, lse);
  a.cap = cap;
  a.slopes = slopes;
  a.out = out;
  if (int rc = check_tree("dilution_tree_softmax", a, length, dtype, d)) return rc;
  if (!out || !scratch || misaligned({scratch})) return abi_fail(DILUTION_ERR_ARG, "dilution_tree_softmax: null or misaligned pointer");
  const int rows = group * nodes;
  a.chunks = tree_chunks((int64_t)a.batch * a.kv_heads * tree_row_blocks(rows), tree_keys(a));
  place_scratch(a, scratch, rows, d);
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    using T = decltype(type);
    if (int rc = rows <= 16 ? simt_softmax<T, dim(), 1, true>(a, st) : simt_softmax<T, dim(), 4, true>(a, st)) return rc;
    return join<T, false>(a, d, st);
  });
}

int dilution_tree_dilute(const void* q, const void* k_new, const void* v_new, const void* k_cache, const void* v_cache, int dtype,
                         int64_t batch, int64_t heads, int nodes, int64_t capacity, int64_t length, const int* length_dev, int d,
                         float scale, float eps, const float* committed, const int* parents, int64_t parent_stride, float* lse,
                         void* out, void* scratch, void* stream) {
  tree::Args a = tree_args(q, k_new, v_new, k_cache, v_cache, parents, parent_stride, batch, heads, 1, nodes, capacity, length,
                           length_dev, scale, lse);
  a.committed = committed;
  a.out = out;
  a.eps = eps;
  if (int rc = check_tree("dilution_tree_dilute", a, length, dtype, d)) return rc;
  if (!out || !committed || !scratch || misaligned({scratch}))
    return abi_fail(DILUTION_ERR_ARG, "dilution_tree_dilute: null or misaligned pointer");
  a.chunks = tree_chunks((int64_t)a.batch * a.kv_heads, tree_keys(a));
  place_scratch(a, scratch, nodes, d);
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    using T = decltype(type);
    if (int rc = nodes <= 16 ? simt_softmax<T, dim(), 1, false>(a, st) : simt_softmax<T, dim(), 4, false>(a, st)) return rc;
    {
      LaunchMark mark("tree_join_stats", st);
      const int64_t all = (int64_t)a.batch * a.kv_heads * nodes;
      tree::join_stats_kernel<<<(unsigned)((all + 7) / 8), 256, 0, st>>>(a);
      if (int rc = abi_check_launch("tree_join_stats")) return rc;
    }
    if (int rc = nodes <= 16 ? simt_dilute<T, dim(), 1>(a, st) : simt_dilute<T, dim(), 4>(a, st)) return rc;
    return join<T, true>(a, d, st);
  });
}

int dilution_tree_accept(const void* q, const void* k_new, const void* v_new, void* k_cache, void* v_cache, int dtype,
                         int64_t batch, int64_t kv_heads, int group, int nodes, int64_t capacity, int64_t length,
                         const int* length_dev, int d, float scale, float cap, const float* slopes, const int* parents,
                         int64_t parent_stride, const float* lse, const int* path, int64_t path_stride, int accepted,
                         const float* committed, float* advanced, void* stream) {
  tree::Args a = tree_args(q, k_new, v_new, k_cache, v_cache, parents, parent_stride, batch, kv_heads, group, nodes, capacity,
                           length, length_dev, scale, const_cast<float*>(lse));
  a.cap = cap;
  a.slopes = slopes;
  a.committed = committed;
  if (int rc = check_tree("dilution_tree_accept", a, length, dtype, d)) return rc;
  if (!path || (committed == nullptr) != (advanced == nullptr)) return abi_fail(DILUTION_ERR_ARG, "dilution_tree_accept: null pointer");
  if (accepted < 1 || accepted > nodes || (!length_dev && length + accepted > capacity))
    return abi_fail(DILUTION_ERR_ARG, "dilution_tree_accept: %d accepted nodes of %d behind %lld keys of %lld", accepted, nodes,
                    (long long)length, (long long)capacity);
  const tree::Accept c{path, path_stride, accepted, advanced, k_cache, v_cache};
  a.chunks = tree_chunks((int64_t)a.batch * a.kv_heads, tree_keys(a));
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    using T = decltype(type);
    if (advanced)
      if (int rc = group * accepted <= 16 ? simt_advance<T, dim(), 1>(a, c, st) : simt_advance<T, dim(), 4>(a, c, st)) return rc;
    LaunchMark mark("tree_append", st);
    const int row_bytes = d * (int)sizeof(T);
    const int64_t threads = (int64_t)a.batch * a.kv_heads * accepted * (row_bytes / 16);
    tree::append_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a, c, row_bytes);
    return abi_check_launch("tree_append");
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
  if (new_capacity < keep || new_capacity > (1 << 30) || n * new_capacity * per / 256 >= (int64_t)1 << 31)
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: new capacity %lld", (long long)new_capacity);
  if (!k_cache || !v_cache || !scores || !k_out || !v_out || !index || (committed == nullptr) != (committed_out == nullptr))
    return abi_fail(DILUTION_ERR_ARG, "dilution_evict: null pointer");
  if (misaligned({k_cache, v_cache, k_out, v_out})) return abi_fail(DILUTION_ERR_ARG, "dilution_evict: caches must be 16-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  {
    // CTAs of a row: until all SMs have one, or a CTA has 1024 keys
    int ranks = 1;
    while (ranks < 8 && n * ranks < 148 && length / (2 * ranks) >= 1024) ranks *= 2;
    while (ranks < 8 && (length + ranks - 1) / ranks > 8192) ranks *= 2;
    evict::Args a;
    a.scores = scores;
    a.score_stride = score_stride;
    a.length = (int)length;
    a.keep = (int)keep;
    a.recent = (int)recent;
    a.sinks = (int)sinks;
    a.seg = (int)((length + ranks - 1) / ranks);
    a.held = a.seg <= evict::kMaxHeld;
    a.index = index;
    const int smem = a.held ? a.seg * 4 : 0;
    if (int rc = opt_in(evict::select_kernel, evict::kMaxHeld * 4)) return rc;
    LaunchMark mark("evict_select", st);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(n * ranks));
    cfg.blockDim = dim3(evict::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, evict::select_kernel, a, ranks);
    if (e != cudaSuccess) return abi_fail(DILUTION_ERR_CUDA, "evict_select: %s", cudaGetErrorString(e));
  }
  LaunchMark mark("evict_gather", st);
  const int64_t threads = n * new_capacity * per;
  evict::gather_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(
      (const uint4*)k_cache, (const uint4*)v_cache, committed, index, n, capacity, (int)keep, new_capacity, per, (uint4*)k_out,
      (uint4*)v_out, committed_out);
  return abi_check_launch("evict_gather");
}

}  // extern "C"
