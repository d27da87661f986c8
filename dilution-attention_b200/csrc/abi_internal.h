// What the translation units of libdilution_b200.so share (host code).
#pragma once

#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/dilution_b200.h"
#include "once_per_device.cuh"

namespace dil {

// Record an error for dilution_last_error() and return its code.
int abi_fail(int code, const char* fmt, ...);
// DILUTION_OK, or the error of the launch in front of it.
int abi_check_launch(const char* what);
// Accounts for one launch (and times it, where that is on) from its construction to its end.
class LaunchMark {
 public:
  LaunchMark(const char* name, cudaStream_t st);
  ~LaunchMark();
  LaunchMark(const LaunchMark&) = delete;
  LaunchMark& operator=(const LaunchMark&) = delete;

 private:
  void* prof_;
};
// The first bounded wait that ran out in a kernel of operators.cu or trees.cu (0: none), read and cleared.  Non-zero: could not
// be read.
int operators_read_status(int* code);
int trees_read_status(int* code);
template <typename W> int read_status_word(const W& word, int* code) {
  int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&v, word, sizeof(int)) != cudaSuccess) return 3;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(word, &zero, sizeof(int));
  }
  *code = v;
  return 0;
}

inline bool valid_d(int d) { return d == 16 || d == 32 || d == 64 || d == 128; }
// A cap of the scores, or 0 for none: what it divides and multiplies stays inside fp32.
inline bool valid_cap(float cap) { return cap == 0.f || (cap >= 1e-30f && cap <= 1e38f); }
inline bool misaligned(std::initializer_list<const void*> ps) {
  uintptr_t x = 0;
  for (const void* p : ps) x |= (uintptr_t)p;
  return x & 15;
}

// Dynamic shared memory (next to `fixed` bytes of a kernel's own) past 48 KB has to be asked for, once per kernel and device.
template <typename K> int opt_in(K kernel, int bytes, int fixed = 0) {
  static OncePerDevice done;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  if (bytes + fixed <= 48 * 1024 || done.done((const void*)kernel, dev)) return DILUTION_OK;
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

// Launch a kernel that may start while the one in front of it in the stream ends (and waits for it itself: wait_for_last).
template <typename... P, typename... A>
int launch_early(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st, const char* name, const A&... args) {
  LaunchMark mark(name, st);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? DILUTION_OK : abi_fail(DILUTION_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

}  // namespace dil
