// The driver's encoder of tensor maps, and what it needs (host code only).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace dil {
namespace tc {

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// The encoder wants a current context, which a thread that has only selected a device (one of autograd's) need not have yet: a
// runtime call that touches the device binds the primary one.  A thread that has a context may be recording a graph, where
// cudaFree is not allowed.
inline void bind_context() {
  static thread_local bool bound = false;
  if (bound) return;
  typedef CUresult (*GetCurrent)(CUcontext*);
  void* get = nullptr;
  cudaDriverEntryPointQueryResult found;
  CUcontext current = nullptr;
  if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &get, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess ||
      ((GetCurrent)get)(&current) != CUDA_SUCCESS || current == nullptr)
    cudaFree(nullptr);
  bound = true;
}

}  // namespace tc
}  // namespace dil
