// Host side of tiled TMA copies: tensor maps. Encoding is a driver call without a stub to link against, found at run time.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace gdn2 {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Encoding needs the device's context to be the thread's own, which a thread that has made no runtime call yet (an autograd
// engine's) lacks. Called before the first map of an entry point.
inline int own_context() {
  int dev = 0;
  GDN2_CUDA_TRY(cudaGetDevice(&dev));
  GDN2_CUDA_TRY(cudaSetDevice(dev));
  return GDN2_OK;
}

}  // namespace gdn2
