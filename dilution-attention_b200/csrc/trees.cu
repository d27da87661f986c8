// extern "C" entry points of draft trees over a cache.  Argument validation, kernel selection and launches; declarations in
// include/dilution_b200.h.

#include <algorithm>
#include <climits>

#include "abi_internal.h"
#include "tc_tree.cuh"
#include "tree_join.cuh"
#include "tree_simt.cuh"

namespace dil {

int trees_read_status(int* code) { return read_status_word(tc::g_tree_status, code); }

namespace {

// Parts that a key head's keys are cut into.  fp32 FMAs: enough blocks for four on every SM, of 128 keys at least.
int simt_chunks(int64_t blocks, int64_t keys) {
  const int64_t want = (148 * 4 + blocks - 1) / std::max<int64_t>(blocks, 1), most = (keys + 127) / 128;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, 512}));
}
// Tensor cores: as many parts as make the fewest rounds of tiles of 128 keys on the chip's SMs, where a block's start and end take as
// long as about four tiles.
int tc_chunks(int64_t blocks, int64_t keys, int per_sm) {
  const int64_t slots = 148 * per_sm;
  const int64_t tiles = std::max<int64_t>(1, (keys + 127) / 128);
  int64_t best = 0;
  int chunks = 1;
  for (int64_t c = 1; c <= std::min<int64_t>(tiles, 2 * 148); ++c) {
    const int64_t cost = (blocks * c + slots - 1) / slots * ((tiles + c - 1) / c + 4);
    if (c == 1 || cost < best) {
      best = cost;
      chunks = (int)c;
    }
  }
  return chunks;
}
int row_blocks(int rows, int of) { return (rows + of - 1) / of; }
int simt_row_blocks(int rows) { return row_blocks(rows, 64); }

template <typename T, int D> constexpr bool kOnTensorCores = std::is_same<T, __nv_bfloat16>::value && (D == 64 || D == 128);

struct TreeScratch {
  size_t part, psum, shares, pout, bytes;
};
TreeScratch tree_scratch(int64_t heads, int group, int nodes, int64_t chunks, int d) {
  TreeScratch s;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t n = (size_t)heads * group * nodes * chunks;
  s.part = 0;
  s.psum = up(n * sizeof(float2));
  s.shares = s.psum + up(n * sizeof(float));
  s.pout = s.shares + up((size_t)heads * nodes * nodes * sizeof(float));
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
  if (!valid_cap(a.cap) || !(a.scale > 0.f))
    return abi_fail(DILUTION_ERR_ARG, "%s: scale must be positive and cap in [1e-30, 1e38], or 0 for none", fn);
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

float* place_scratch(tree::Args& a, void* scratch, int d) {
  const TreeScratch s = tree_scratch((int64_t)a.batch * a.kv_heads, a.group, a.nodes, a.chunks, d);
  char* p = (char*)scratch;
  a.part = (float2*)(p + s.part);
  a.psum = (float*)(p + s.psum);
  a.pout = (float*)(p + s.pout);
  return (float*)(p + s.shares);
}

// f(integral_constant<int, RI>()): the fewest rows of 16 that hold `rows` of them, four at most.
template <typename F> int with_rows(int rows, F f) {
  if (rows <= 16) return f(std::integral_constant<int, 1>());
  if (rows <= 32) return f(std::integral_constant<int, 2>());
  if (rows <= 48) return f(std::integral_constant<int, 3>());
  return f(std::integral_constant<int, 4>());
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

// ---- tensor cores
int cache_maps(CUtensorMap* k, CUtensorMap* v, const tree::Args& a, int d) {
  const int64_t n = (int64_t)a.batch * a.kv_heads;
  if (!tc::tile_map(k, a.kc, n, a.capacity, d, 64) || !tc::tile_map(v, a.vc, n, a.capacity, d, 64))
    return abi_fail(DILUTION_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  return DILUTION_OK;
}

template <int D, int G, bool OUT> int tc_scan_rows(const tree::Args& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  using F = tc::Scan<D, G, OUT>;
  if (int rc = opt_in(tc::scan_kernel<D, G, OUT>, F::kBytes)) return rc;
  LaunchMark mark(OUT ? "tree_softmax" : "tree_stats", st);
  const dim3 grid(a.chunks, G == 1 ? row_blocks(a.group * a.nodes, 128) : 1, a.batch * a.kv_heads);
  tc::scan_kernel<D, G, OUT><<<grid, F::kThreads, F::kBytes, st>>>(k, v, a);
  return abi_check_launch("tree_scan");
}
template <int D, bool OUT> int tc_scan(const tree::Args& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  const int rows = a.group * a.nodes;
  if (rows <= 32) return tc_scan_rows<D, 4, OUT>(a, k, v, st);
  if (rows <= 64) return tc_scan_rows<D, 2, OUT>(a, k, v, st);
  if constexpr (OUT) return tc_scan_rows<D, 1, OUT>(a, k, v, st);
  return DILUTION_OK;            // (a dilution layer's rows are its nodes, 64 at most)
}
template <int D, int N, bool DILUTE>
int tc_sweep_rows(const tree::Args& a, const tree::Accept& c, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  using F = tc::Sweep<D, N, DILUTE>;
  if (int rc = opt_in(tc::sweep_kernel<D, N, DILUTE>, F::kBytes)) return rc;
  const dim3 grid(a.chunks, 1, a.batch * a.kv_heads);
  if (DILUTE) return launch_early(tc::sweep_kernel<D, N, DILUTE>, grid, F::kThreads, F::kBytes, st, "tree_dilute", k, v, a, c);
  LaunchMark mark("tree_advance", st);
  tc::sweep_kernel<D, N, DILUTE><<<grid, F::kThreads, F::kBytes, st>>>(k, v, a, c);
  return abi_check_launch("tree_advance");
}
template <int D, bool DILUTE>
int tc_sweep(const tree::Args& a, const tree::Accept& c, int rows, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  if (rows <= 16) return tc_sweep_rows<D, 16, DILUTE>(a, c, k, v, st);
  if (rows <= 32) return tc_sweep_rows<D, 32, DILUTE>(a, c, k, v, st);
  return tc_sweep_rows<D, 64, DILUTE>(a, c, k, v, st);
}

template <int D> int tc_softmax(tree::Args a, void* scratch, cudaStream_t st) {
  CUtensorMap k, v;
  if (int rc = cache_maps(&k, &v, a, D)) return rc;
  const int rows = a.group * a.nodes;
  a.chunks = tc_chunks((int64_t)a.batch * a.kv_heads * row_blocks(rows, 128), tree_keys(a), tc::Scan<D, 4, true>::kPerSm);
  place_scratch(a, scratch, D);
  if (int rc = tc_scan<D, true>(a, k, v, st)) return rc;
  if (int rc = opt_in(tree::join_softmax_kernel<D>, tree::join_softmax_smem<D>(tree::kMaxNodes))) return rc;
  return launch_early(tree::join_softmax_kernel<D>, dim3((unsigned)((int64_t)a.batch * a.kv_heads * a.group)), tree::join_threads(a.nodes),
                      tree::join_softmax_smem<D>(a.nodes), st, "tree_join", a);
}

// A step in one launch, a cluster of eight CTAs per head: for short caches whose clusters all run at once (a CTA of heads of 128 has an
// SM to itself, and clusters of them do not share one).  24 nodes, one launch / chunks (four launches that start early), both replayed from
// a graph, us.  Heads of 64: 1 head, 1024 keys 25 / 29, 8192 keys 35 / 33; 8 heads, 1024 27 / 31, 8192 37 / 41; 16 heads, 1024 29 / 35, 8192
// 41 / 41, 16384 57 / 51; 32 heads, 1024 30 / 37, 8192 45 / 53; 64 heads, 4096 64 / 51.  Heads of 128: 1 head, 1024 29 / 31, 8192 43 / 35;
// 8 heads, 1024 29 / 33, 4096 35 / 35; 16 heads, 512 51 / 33; 32 heads, 8192 115 / 66.
template <int D> bool by_clusters(const tree::Args& a) {
  return (int64_t)a.batch * a.kv_heads <= (D == 64 ? 32 : 8) && tree_keys(a) <= (D == 64 ? 8192 : 4096) + tree::kMaxNodes;
}
template <int D, int N> int tc_draft(const tree::Args& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  using F = tc::Draft<D, N>;
  if (int rc = opt_in(tc::draft_kernel<D, N>, F::kBytes)) return rc;
  LaunchMark mark("tree_draft", st);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = tc::kDraftRanks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(a.batch * a.kv_heads * tc::kDraftRanks));
  cfg.blockDim = dim3(F::kThreads);
  cfg.dynamicSmemBytes = F::kBytes;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tc::draft_kernel<D, N>, k, v, a);
  return e == cudaSuccess ? DILUTION_OK : abi_fail(DILUTION_ERR_CUDA, "tree_draft: %s", cudaGetErrorString(e));
}

template <int D> int tc_dilute(tree::Args a, void* scratch, cudaStream_t st) {
  CUtensorMap k, v;
  if (int rc = cache_maps(&k, &v, a, D)) return rc;
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  if (by_clusters<D>(a)) return a.nodes <= 16 ? tc_draft<D, 16>(a, k, v, st) : a.nodes <= 32 ? tc_draft<D, 32>(a, k, v, st) : tc_draft<D, 64>(a, k, v, st);
  a.chunks = tc_chunks(heads, tree_keys(a), tc::Sweep<D, 64, true>::kPerSm);
  float* shares = place_scratch(a, scratch, D);
  if (int rc = tc_scan<D, false>(a, k, v, st)) return rc;
  if (int rc = opt_in(tree::join_bids_kernel<D>, 64 * 65 * 4, 36 * 1024)) return rc;
  if (int rc = launch_early(tree::join_bids_kernel<D>, dim3((unsigned)heads), tree::join_threads(a.nodes), a.nodes * (a.nodes + 1) * 4, st,
                            "tree_join_bids", a, shares)) return rc;
  if (int rc = tc_sweep<D, true>(a, tree::Accept{}, a.nodes, k, v, st)) return rc;
  return launch_early(tree::join_dilute_kernel<D>, dim3((unsigned)(heads * a.nodes)), D, 0, st, "tree_join", a, shares);
}

template <int D> int tc_accept(tree::Args a, const tree::Accept& c, cudaStream_t st) {
  if (c.advanced) {
    CUtensorMap k, v;
    if (int rc = cache_maps(&k, &v, a, D)) return rc;
    a.chunks = tc_chunks((int64_t)a.batch * a.kv_heads, tree_keys(a), 2);
    if (int rc = tc_sweep<D, false>(a, c, a.group * c.accepted, k, v, st)) return rc;
  }
  // (it starts early behind the sweep alone: what it reads in front of its wait may be another kernel's work otherwise)
  if (c.advanced) return launch_early(tree::accept_nodes_kernel<D>, dim3((unsigned)(a.batch * a.kv_heads)), 256, 0, st, "tree_append", a, c);
  LaunchMark mark("tree_append", st);
  tree::accept_nodes_kernel<D><<<(unsigned)(a.batch * a.kv_heads), 256, 0, st>>>(a, c);
  return abi_check_launch("tree_append");
}

}  // namespace
}  // namespace dil

using namespace dil;

extern "C" {

size_t dilution_tree_scratch_bytes(int64_t batch, int64_t kv_heads, int group, int nodes, int64_t length, int d) {
  if (batch < 1 || kv_heads < 1 || group < 1 || nodes < 1 || length < 0 || d < 1) return 0;
  const int64_t heads = batch * kv_heads, keys = length + nodes;
  const int rows = group * nodes;
  const int chunks = std::max(simt_chunks(heads * simt_row_blocks(rows), keys), std::max(tc_chunks(heads * row_blocks(rows, 128), keys, 1), tc_chunks(heads * row_blocks(rows, 128), keys, 2)));
  return tree_scratch(heads, group, nodes, chunks, d).bytes;
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
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    using T = decltype(type);
    if constexpr (kOnTensorCores<T, dim()>) return tc_softmax<dim()>(a, scratch, st);
    else {
    a.chunks = simt_chunks((int64_t)a.batch * a.kv_heads * simt_row_blocks(rows), tree_keys(a));
    place_scratch(a, scratch, d);
    if (int rc = with_rows(rows, [&](auto ri) { return simt_softmax<T, dim(), ri(), true>(a, st); })) return rc;
    return join<T, false>(a, d, st);
    }
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
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    using T = decltype(type);
    if constexpr (kOnTensorCores<T, dim()>) return tc_dilute<dim()>(a, scratch, st);
    else {
    a.chunks = simt_chunks((int64_t)a.batch * a.kv_heads * simt_row_blocks(nodes), tree_keys(a));
    place_scratch(a, scratch, d);
    if (int rc = with_rows(nodes, [&](auto ri) { return simt_softmax<T, dim(), ri(), false>(a, st); })) return rc;
    {
      LaunchMark mark("tree_join_stats", st);
      const int64_t all = (int64_t)a.batch * a.kv_heads * nodes;
      tree::join_stats_kernel<<<(unsigned)((all + 7) / 8), 256, 0, st>>>(a);
      if (int rc = abi_check_launch("tree_join_stats")) return rc;
    }
    if (int rc = with_rows(nodes, [&](auto ri) { return simt_dilute<T, dim(), ri()>(a, st); })) return rc;
    return join<T, true>(a, d, st);
    }
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
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(dtype, d, [&](auto type, auto dim) {
    using T = decltype(type);
    if constexpr (kOnTensorCores<T, dim()>)
      if (!advanced || group * accepted <= 64) return tc_accept<dim()>(a, c, st);
    a.chunks = simt_chunks((int64_t)a.batch * a.kv_heads, tree_keys(a));
    if (advanced)
      if (int rc = group * accepted <= 16 ? simt_advance<T, dim(), 1>(a, c, st) : simt_advance<T, dim(), 4>(a, c, st)) return rc;
    LaunchMark mark("tree_append", st);
    const int row_bytes = d * (int)sizeof(T);
    const int64_t threads = (int64_t)a.batch * a.kv_heads * accepted * (row_bytes / 16);
    tree::append_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a, c, row_bytes);
    return abi_check_launch("tree_append");
  });
}

}  // extern "C"
