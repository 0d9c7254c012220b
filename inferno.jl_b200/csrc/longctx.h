// Host-side helpers shared by the long-context operators (rope.cu,
// attn_cached.cu, evict.cu).
#pragma once
#include <cuda_runtime.h>
#include "internal.h"
#include "../../include/inferno_b200.h"

namespace inf {

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994)
struct FastDiv {
  uint32_t d, mul, shift;
  __host__ FastDiv(uint32_t div = 1) : d(div) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// bytes of an element of the operators' types, 0 for any other type
inline int longctx_type_size(int type) {
  return type == INFERNO_F32 ? 4 : type == INFERNO_F16 || type == INFERNO_BF16 ? 2 : 0;
}

// A launch goes to the current device: refuse a buffer that lives on another
// one, or that the device cannot reach, before a kernel faults on it.
inline int longctx_check_device(const void* p, const char* what) {
  cudaPointerAttributes at{};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaPointerGetAttributes(&at, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(INFERNO_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  if (at.type == cudaMemoryTypeUnregistered)
    return set_error(INFERNO_EINVAL, "%s: an output is not device memory", what);
  if (at.type == cudaMemoryTypeDevice && at.device != dev)
    return set_error(INFERNO_EINVAL, "%s: buffers are on device %d, the current device is %d", what, at.device, dev);
  return 0;
}

}  // namespace inf
