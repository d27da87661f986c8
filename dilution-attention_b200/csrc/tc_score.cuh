// What the tensor-core kernels of the operators around the attention layers share: scores through a cap, packing, and
// tensor maps.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"
#include "tensor_maps.cuh"

namespace dil {
namespace tc {

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float2 unpack_pair(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
// What the rounding of such a pair leaves off.
__device__ __forceinline__ uint32_t left_pair(float lo, float hi) {
  const float2 r = unpack_pair(pack_pair(lo, hi));
  return pack_pair(lo - r.x, hi - r.y);
}

// Head sizes: D / 64 sub-tiles of 64 features (tc_common.cuh).
template <int D> constexpr int kForm = D == 128 ? kWide128 : kNarrow;

// ---- scores ----------------------------------------------------------------------------------------
// tanh of two values, |x| <= 1 (tanh_score).  Nine packed instructions, where the two special-function operations of a value take 16
// cycles of a warp's quarter.
__device__ __forceinline__ float2 tanh_poly2(float2 x) {
  auto both = [](float c) { return make_float2(c, c); };
  const float2 y = mul2(x, x);
  float2 p = both(kTanh[5]);
#pragma unroll
  for (int i = 4; i >= 0; --i) p = fma2(p, y, both(kTanh[i]));
  p = mul2(p, y);
  return fma2(x, p, x);
}
// v = tanh(v * pre) of N products q . k.  pre: scale / cap.  Where a score of the warp is past the cap all take the form for those, which
// is off by 4e-7 of the cap: at most 4e-4 of a score up to caps of 1024, a tenth of what the rounding of P~ may be.  wide: larger
// caps, each score by its own size.  (That for all caps: B2 H16 T8192, heads of 128, scores past a cap of 5, forward 1087 -> 1830 us.)
template <int N> __device__ __forceinline__ void cap_scores(float* v, float pre, bool wide) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < N; e += 2) top = fmaxf(top, fmaxf(fabsf(v[e]), fabsf(v[e + 1])));
  // (fmaxf passes over a NaN, which comes through either form)
  if (!__any_sync(0xffffffffu, top * pre > 1.f)) {
    const float2 pp = make_float2(pre, pre);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 t = tanh_poly2(mul2(make_float2(v[e], v[e + 1]), pp));
      v[e] = t.x;
      v[e + 1] = t.y;
    }
  } else if (wide) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = tanh_score(v[e] * pre);
  } else {
    const float twice = pre * 2.f * kLog2e;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = fmaf(-2.f, fast_rcp(1.f + fast_exp2(v[e] * twice)), 1.f);
  }
}
constexpr float kWideCap = 1024.f;

// ---- tensor maps -----------------------------------------------------------------------------------
// (n, t, d) bf16 rows as boxes {64 features, box rows, 1}, 128-byte swizzle; rows past t read as zero.  True: encoded.
inline bool tile_map(CUtensorMap* map, const void* base, int64_t n, int64_t t, int d, int box) {
  bind_context();
  EncodeTiled fn = encode_tiled();
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)t, (cuuint64_t)n};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)t * d * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)box, 1}, ones[3] = {1, 1, 1};
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, boxes, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
}  // namespace dil
