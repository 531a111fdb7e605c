// Dynamic shared memory beyond the default 48 KB.
#pragma once

#include <cuda_runtime_api.h>
#include <stddef.h>

#include <exception>
#include <map>
#include <mutex>
#include <utility>

namespace ckv {

// Opt a kernel in to `bytes` of dynamic shared memory on the current device.  The attribute is per
// kernel and device and only ever raised (a smaller request never lowers it under a larger launch
// issued elsewhere).
inline cudaError_t ensure_dynamic_smem(const void* func, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, size_t> have;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
  try {
    std::lock_guard<std::mutex> lock(mu);
    size_t& h = have[{device, func}];
    if (bytes <= h) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) h = bytes;
    return e;
  } catch (const std::exception&) {   // the map's memory or the lock: no exception leaves a C entry
    return cudaErrorMemoryAllocation;
  }
}

}  // namespace ckv
