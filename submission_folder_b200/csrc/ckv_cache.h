// Launch interface of the paged 8-bit decode cache: block tables, rotary positions,
// cache write / read, attention over the cache.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/ckv.h"

namespace ckv {

// A launch that may begin while the launch before it on the stream drains (programmatic
// dependent launch): its blocks are placed early and wait in after_previous(), which every
// kernel launched so calls in every thread before it touches global memory.  Saves the gap
// between the short kernels of a decode step.  What the launch before may have written is read
// with plain loads only: read-only (non-coherent) ones are defined for data that is constant while
// the kernel is resident, and neither those nor cache-hinted ones are bound to stay behind the wait.
template <typename... P>
cudaError_t launch_after(void (*fn)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, P... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, args...);
}
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the next launch may be placed
  asm volatile("griddepcontrol.wait;" ::: "memory");                // the previous one is complete
}

constexpr int kMaxRequests = 8192;   // rows of one block-table step (their prefix sums sit in shared memory)
constexpr int kCacheMaxBlock = 128;  // tokens of a cache block: 16, 32, 64 or 128

cudaError_t launch_block_tables(const ckv_table_step& s, cudaStream_t st);

cudaError_t launch_rotary(const ckv_rotary_args& a, cudaStream_t st);

struct CacheRows {          // token rows [tokens][heads][D] of keys and values
  void* k;
  int64_t kts, khs;         // strides in elements
  void* v;
  int64_t vts, vhs;
  int dtype;
  const int64_t* slots;     // [tokens]: block * block_size + offset; anything outside the pool is no token
  int tokens;
};
cudaError_t launch_cache_write(const ckv_cache& c, const CacheRows& r, cudaStream_t st);
cudaError_t launch_cache_read(const ckv_cache& c, const CacheRows& r, cudaStream_t st);

size_t attention_workspace_bytes(int head_dim, int rows);
cudaError_t launch_cache_attention(const ckv_cache& c, const ckv_attention_args& a, void* ws, cudaStream_t st);

}  // namespace ckv
