// Launch interface of the paged 8-bit decode cache: block tables, rotary positions,
// cache write / read, attention over the cache.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/ckv.h"

namespace ckv {

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
