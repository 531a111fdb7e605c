// How the stores of one request of a large block-table step are shared out.  Plain C++, so that
// the host can check the arithmetic at the ends of its range.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define CKV_SHARE_FN __host__ __device__ __forceinline__
#else
#define CKV_SHARE_FN inline
#endif

namespace ckv {

struct Share {
  uint32_t from, to;   // tokens of the request
};

// Part `part` of `parts` (at most 64) of a request's tokens.  granted > 0: all of those, whose table
// entries are written whether or not the step has a row for them.  Otherwise the `asked` tokens of a
// refused request, or of one that has none, as far as the step's rows go: `total` rows, the request's
// first at t0.  asked, t0 and total are at most 2^31 - 1, so a loop from `from` by steps of a CTA's
// threads stays below 2^32.
CKV_SHARE_FN Share share_of(int32_t asked, int32_t granted, int32_t t0, int32_t total, int32_t part, int32_t parts) {
  const uint32_t rows = total > t0 ? (uint32_t)(total - t0) : 0u;
  const uint32_t n = granted > 0 ? (uint32_t)granted : (uint32_t)asked < rows ? (uint32_t)asked : rows;
  const uint32_t each = n / parts + (n % parts ? 1u : 0u), at = part * each, end = at + each;
  return {at < n ? at : n, end < n ? end : n};
}

}  // namespace ckv
