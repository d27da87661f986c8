// Sums over many rows by one warp, for what the tile kernels leave over.  A lane has 16 bytes of a row, so that a warp has several
// rows at once, kSteps times; each group of lanes that share a row keeps sums of its own, which are joined at the end.
#pragma once

#include "common.cuh"

namespace dil {

template <typename T, int D> struct Lanes {
  static constexpr int E = 16 / (int)sizeof(T), L = D / E, R = 32 / L;      // elements of a lane, lanes of a row, rows at once
  static constexpr int kSteps = 4, kRows = R * kSteps;
  int part, own;                                                            // the lane's elements, its row
  __device__ __forceinline__ Lanes() : part((int)(threadIdx.x & 31) % L), own((int)(threadIdx.x & 31) / L) {}
  __device__ __forceinline__ uint4 load(const T* rows, int row) const {
    return reinterpret_cast<const uint4*>(rows + (int64_t)row * D)[part];
  }
  __device__ __forceinline__ float of(const uint4& u, int e) const { return to_f32(reinterpret_cast<const T*>(&u)[e]); }
  // x . y, in each of a row's lanes
  __device__ __forceinline__ float dot(const uint4& x, const uint4& y) const {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(of(x, e), of(y, e), s);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
  static __device__ __forceinline__ float over_rows(float s) {
#pragma unroll
    for (int o = L; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
  static __device__ __forceinline__ float max_over_rows(float m) {
#pragma unroll
    for (int o = L; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
};
template <typename T, int D> struct LaneSums : Lanes<T, D> {
  using B = Lanes<T, D>;
  float x[B::E] = {};
  __device__ __forceinline__ void scale(float f) {
#pragma unroll
    for (int e = 0; e < B::E; ++e) x[e] *= f;
  }
  __device__ __forceinline__ void add(float f, const uint4& u) {
#pragma unroll
    for (int e = 0; e < B::E; ++e) x[e] = fmaf(f, this->of(u, e), x[e]);
  }
  // No feature of the row is a number any more.
  __device__ __forceinline__ bool no_number() const {
    unsigned bits = 0;
#pragma unroll
    for (int e = 0; e < B::E; ++e) bits |= (x[e] != x[e] ? 1u : 0u) << e;
#pragma unroll
    for (int o = B::L; o < 32; o <<= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, o);
    return __all_sync(0xffffffffu, bits == (1u << B::E) - 1);
  }
  __device__ __forceinline__ void join(float f) {
#pragma unroll
    for (int e = 0; e < B::E; ++e) x[e] = B::over_rows(x[e]) * f;
  }
  __device__ __forceinline__ void store(T* p) const {
    uint4 u;
#pragma unroll
    for (int e = 0; e < B::E; ++e) reinterpret_cast<T*>(&u)[e] = from_f32<T>(x[e]);
    if (this->own == 0) reinterpret_cast<uint4*>(p)[this->part] = u;
  }
};

}  // namespace dil
