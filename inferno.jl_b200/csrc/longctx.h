// Host-side helpers shared by the long-context operators (rope.cu,
// attn_cached.cu, evict.cu).
#pragma once
#include <initializer_list>
#include <cuda.h>
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

// A launch goes to the current device: refuse any buffer (nulls are passed over) that
// lives on another one, or that is no memory of CUDA's, before a kernel faults on it.
// The driver's one attribute takes 28 ns a buffer; the runtime's record of all of them,
// 65 ns, is asked for only where that does not settle it.
inline int longctx_check_device(std::initializer_list<const void*> buffers, const char* what) {
  using Get = CUresult (*)(void*, CUpointer_attribute, CUdeviceptr);
  static const Get get = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuPointerGetAttribute", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (Get)p;
  }();
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  for (const void* p : buffers) {
    if (!p || e != cudaSuccess) continue;
    int at_dev = -1;
    if (get && get(&at_dev, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, (CUdeviceptr)p) == CUDA_SUCCESS && at_dev == dev) continue;
    cudaPointerAttributes at{};
    e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) continue;
    if (at.type == cudaMemoryTypeUnregistered)
      return set_error(INFERNO_EINVAL, "%s: a buffer is not device memory", what);
    if (at.type == cudaMemoryTypeDevice && at.device != dev)
      return set_error(INFERNO_EINVAL, "%s: a buffer is on device %d, the current device is %d", what, at.device, dev);
  }
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  return set_error(INFERNO_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace inf
