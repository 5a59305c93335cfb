// Host-side helpers of the entry points over the 8-bit paged cache.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "silkern_b200.h"

namespace silkern {

// Launch `fn` under programmatic dependent launch, `cluster` CTAs to a
// thread-block cluster. 0 or -(cudaError_t).
template <typename... P, typename... A>
int launch_pdl_grid(void (*fn)(P...), dim3 grid, unsigned threads, size_t smem, unsigned cluster,
                    cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attrs;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, fn, args...);
  if (err != cudaSuccess) {
    (void)cudaGetLastError();
    return -static_cast<int>(err);
  }
  return SILKERN_OK;
}

template <typename... P, typename... A>
int launch_pdl(void (*fn)(P...), unsigned grid, unsigned threads, size_t smem, unsigned cluster,
               cudaStream_t stream, A&&... args) {
  return launch_pdl_grid(fn, dim3(grid, 1, 1), threads, smem, cluster, stream, args...);
}

// Devices that `known` notes of a kernel's launch permissions; others are asked
// for at each call. Nothing here allocates or throws: C callers come in.
constexpr int kNotedDevices = 64;
using DeviceBits = std::atomic<uint64_t>;

// Let `kernel` use `bytes` of dynamic shared memory, all of an SM's shared
// memory, and clusters of up to 16 CTAs, on the current device. The driver is
// asked once for each kernel (which has a `granted` of its own) and device.
inline int allow_launch(const void* kernel, int bytes, DeviceBits& granted) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess) {
    const uint64_t bit = device < kNotedDevices ? uint64_t{1} << device : 0;
    if ((granted.load(std::memory_order_acquire) & bit) != 0) return SILKERN_OK;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess) {
      err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
    if (err == cudaSuccess) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err == cudaSuccess) granted.fetch_or(bit, std::memory_order_release);
  }
  if (err == cudaSuccess) return SILKERN_OK;
  (void)cudaGetLastError();
  return -static_cast<int>(err);
}

}  // namespace silkern
