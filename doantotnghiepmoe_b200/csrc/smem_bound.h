// The bound on a kernel's dynamic shared memory.
//
// It belongs to the kernel (on a device), which every handle and every host
// thread of the process launches, and a launch that takes more is refused.  A
// launcher whose need depends on the call therefore only ever raises it: set to
// a call's own need, it would refuse the launches of another handle with wider
// layers, between that handle's own setting and its launch, or for good where a
// launcher sets it once per thread.
#pragma once

#include <algorithm>
#include <cstddef>
#include <map>
#include <mutex>
#include <utility>

#include <cuda_runtime.h>

namespace moe {

// Kernel fn may be launched with `bytes` on the current device.
inline cudaError_t allow_smem(const void *fn, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void *>, size_t> most;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  size_t &m = most[{dev, fn}];
  m = std::max(m, bytes);
  return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)m);
}

}  // namespace moe
