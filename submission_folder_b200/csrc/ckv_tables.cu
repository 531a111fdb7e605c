// Block tables, slots and positions of one decode / admission step, from the requests'
// lengths, on the device: a step of a captured graph can admit, extend and end requests
// without the host.
//
// With b tokens per block, request r holds ceil(len / b) blocks and needs
// ceil((len + new) / b) - ceil(len / b) more; new < 0 ends it and gives its blocks back.
// The free blocks are a stack.  Blocks given back go on top (requests in order, blocks in
// order); fresh blocks come off the top (requests in order, blocks in order).  All of it is
// three prefix sums over the requests (tokens, blocks back, blocks needed); after them each
// token and each block finds its request by binary search and its block by arithmetic on the
// sums, independently of all others (a block that is given back and taken in the same step is
// looked up where it was given back, not where it is put down).
//
// Bound: latency.  A small step is one CTA: scan, then stores, each token's request found by
// binary search in shared memory.  Above CKV_TABLES_SMALL tokens and requests the stores go to a second
// launch with CTAs for each request, which need no search but for blocks that came back in the
// same step (1024 requests, 602,000 tokens, kernels alone: 126 us when a cluster of 8 CTAs searched for
// every token, 17 us in two launches that did, 12 with CTAs by request).  16 requests of 500, 2000, 4000 and
// 8000 tokens in all: one CTA 3.5, 4.4, 5.9 and 9.0 us, two launches 4.3 to 4.4; 1000 requests of 1000 and 3000:
// 5.0 and 7.1 against 6.0; 3000 of 1000: 10.2 against 11.7.
#include <algorithm>

#include "ckv_cache.h"
#include "ckv_common.cuh"
#include "ckv_share.h"

namespace ckv {

constexpr int kTabThreads = 1024;

struct Sum3 {
  long long tok;   // requested tokens
  int back, need;  // blocks given back, fresh blocks wanted
};

CKV_DEV Sum3 operator+(const Sum3& x, const Sum3& y) { return {x.tok + y.tok, x.back + y.back, x.need + y.need}; }
CKV_DEV Sum3 shfl_up(const Sum3& x, int o) {
  return {__shfl_up_sync(0xffffffffu, x.tok, o), __shfl_up_sync(0xffffffffu, x.back, o),
          __shfl_up_sync(0xffffffffu, x.need, o)};
}

// Exclusive block scan; *total gets the block's sum.
CKV_DEV Sum3 scan3(Sum3 v, Sum3* scratch, Sum3* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  Sum3 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sum3 y = shfl_up(x, o);
    if (lane >= o) x = x + y;
  }
  __syncthreads();
  if (lane == 31) scratch[wid] = x;
  __syncthreads();
  if (wid == 0) {
    Sum3 s = lane < nw ? scratch[lane] : Sum3{0, 0, 0};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Sum3 y = shfl_up(s, o);
      if (lane >= o) s = s + y;
    }
    scratch[lane] = s;
  }
  __syncthreads();
  const Sum3 base = wid > 0 ? scratch[wid - 1] : Sum3{0, 0, 0};
  *total = scratch[nw - 1];
  return {base.tok + x.tok - v.tok, base.back + x.back - v.back, base.need + x.need - v.need};
}

// Last row in [lo, hi] whose prefix p[row] is <= x (p ascending, p[lo] <= x).
CKV_DEV int row_of(const int* p, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// What the scan leaves for the stores: prefixes over the requests, and per request the old length
// and the tokens granted; the stack's height before (count), with what came back (have), and the
// blocks taken.
struct StepView {
  const int *cu, *back, *fresh, *len, *give;
  int count, have, taken;
};

// Stores of the threads gt of gn: blocks given back, table entries, slots and positions.
CKV_DEV void fill_step(const ckv_table_step& s, const StepView& v, int gt, int gn) {
  const int R = s.requests;
  const uint32_t b = s.block_size;
  // the j-th block from the bottom of the stack, after the blocks given back went on top
  auto stack = [&](int j) -> int {
    if (j < v.count) return s.free_list[j];
    const int e = j - v.count, r = row_of(v.back, 0, R - 1, e);
    return s.tables[r * s.table_stride + (e - v.back[r])];
  };
  for (int i = gt; i < v.have - v.count; i += gn) s.free_list[v.count + i] = stack(v.count + i);
  for (int i = gt; i < v.taken; i += gn) {
    const int r = row_of(v.fresh, 0, R - 1, i);
    s.tables[r * s.table_stride + ((uint32_t)v.len[r] + b - 1) / b + (i - v.fresh[r])] = stack(v.have - 1 - i);
  }
  const int asked = v.cu[R];
  for (int t = gt; t < s.total; t += gn) {
    long long slot = -1, where = 0;
    if (t < asked) {
      const int r = row_of(v.cu, 0, R - 1, t);
      const uint32_t n = v.len[r], pos = n + (uint32_t)(t - v.cu[r]);
      where = (long long)pos + (s.shift ? s.shift[r] : 0);
      if (v.give[r] > 0) {
        const uint32_t bi = pos / b, held = (n + b - 1) / b;
        const int block = bi < held ? s.tables[r * s.table_stride + bi]
                                    : stack(v.have - 1 - (v.fresh[r] + (int)(bi - held)));
        slot = (long long)block * b + (pos - bi * b);
      }
    }
    s.out_slots[t] = slot;
    s.out_positions[t] = where;
  }
}

// The scan, by one CTA; and the stores, when they are few.
__global__ void __launch_bounds__(kTabThreads) k_block_tables(const ckv_table_step s, int solo) {
  extern __shared__ int tab_smem[];
  __shared__ Sum3 scratch[32];
  __shared__ int s_taken;
  const int R = s.requests, b = s.block_size, tid = threadIdx.x;
  int* cu = tab_smem;             // [R + 1] tokens before request r, as asked for
  int* back = cu + R + 1;         // [R + 1] blocks given back before request r
  int* fresh = back + R + 1;      // [R + 1] fresh blocks wanted before request r
  int* len = fresh + R + 1;       // [R] old length
  int* give = len + R;            // [R] tokens granted; before that -2: ended, -1: does not fit its row
  after_previous();
  if (tid == 0) s_taken = 0;
  const int count = min(max(*s.free_count, 0), s.free_capacity);
  Sum3 run = {0, 0, 0};
  for (int base = 0; base < R; base += blockDim.x) {
    const int r = base + tid;
    Sum3 v = {0, 0, 0};
    if (r < R) {
      const int n = max(s.lens[r], 0), nw = s.new_tokens[r];
      const int held = (int)(((uint32_t)n + b - 1) / b);
      len[r] = n;
      if (nw < 0) {
        v.back = min(held, s.table_width);
        give[r] = -2;
      } else {
        v.tok = nw;
        const uint32_t want = (uint32_t)n + nw == 0 ? 0u : ((uint32_t)n + nw - 1) / b + 1;
        const bool fits = want <= (uint32_t)s.table_width && (uint32_t)n + nw <= (uint32_t)INT32_MAX;
        give[r] = fits ? nw : -1;
        v.need = fits ? (int)want - held : 0;
      }
    }
    Sum3 total;
    const Sum3 ex = scan3(v, scratch, &total);
    if (r < R) {
      cu[r] = (int)min(run.tok + ex.tok, (long long)INT32_MAX);
      back[r] = run.back + ex.back;
      fresh[r] = run.need + ex.need;
    }
    run = run + total;
  }
  if (tid == 0) {
    cu[R] = (int)min(run.tok, (long long)INT32_MAX);
    back[R] = run.back;
    fresh[R] = run.need;
  }
  __syncthreads();
  const int have = (int)min((long long)count + run.back, (long long)s.free_capacity);
  for (int r = tid; r < R; r += blockDim.x) {   // fresh blocks go to the requests in order while they last
    const int need = fresh[r + 1] - fresh[r], was = give[r];
    if (was >= 0 && need > 0) {
      if (fresh[r + 1] <= have) atomicMax(&s_taken, fresh[r + 1]);
      else give[r] = -1;
    }
    const int granted = max(give[r], 0);
    const bool refused = was != -2 && give[r] < 0;
    give[r] = granted;
    s.out_cu[r] = cu[r];
    s.out_granted[r] = granted;
    s.out_lens[r] = was == -2 ? 0 : len[r] + granted;
    if (s.out_seen) s.out_seen[r] = was == -2 || refused ? 0 : len[r] + granted;
  }
  __syncthreads();
  const int taken = s_taken;
  if (tid == 0) {
    s.out_cu[R] = cu[R];
    s.out_free_count[0] = have - taken;
  }
  if (solo) {
    fill_step(s, StepView{cu, back, fresh, len, give, count, have, taken}, tid, blockDim.x);
    return;
  }
  int* w = s.work;                // [3 R + 4]: back, fresh, old length, count, have
  for (int i = tid; i <= R; i += blockDim.x) {
    w[i] = back[i];
    w[R + 1 + i] = fresh[i];
    if (i < R) w[2 * (R + 1) + i] = len[i];
  }
  if (tid < 2) w[3 * R + 2 + tid] = tid == 0 ? count : have;
}

// The stores of a large step: CTA (r, part) has a part of request r's tokens, CTA (R, part) of
// the rows past the last request's.
constexpr int kFillThreads = 128, kFillBlocks = 512;

// Last row whose prefix p[row] is <= x, by one warp, 32 probes at a time; p in global memory.
CKV_DEV int warp_row_of(const int* p, int rows, int x) {
  int lo = 0, n = rows;
  while (n > 1) {
    const int step = (n + 31) / 32, i = (threadIdx.x & 31) * step;
    const uint32_t m = __ballot_sync(0xffffffffu, i < n && p[lo + min(i, n - 1)] <= x);
    const int hit = m ? 31 - __clz(m) : 0;
    lo += hit * step;
    n = min(step, n - hit * step);
  }
  return lo;
}

__global__ void __launch_bounds__(kFillThreads) k_block_tables_fill(const ckv_table_step s) {
  __shared__ int s_id[kFillBlocks];
  const int R = s.requests, r = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  const uint32_t b = s.block_size;
  after_previous();
  const int *back = s.work, *fresh = back + R + 1, *len = fresh + R + 1, *tail = len + R;
  if (r == R) {   // no request's tokens
    for (int64_t t = (int64_t)s.out_cu[R] + part * kFillThreads + tid; t < s.total; t += parts * kFillThreads) {
      s.out_slots[t] = -1;
      s.out_positions[t] = 0;
    }
    return;
  }
  const int t0 = s.out_cu[r], ask = s.out_cu[r + 1] - t0, give = s.out_granted[r];
  const int n = len[r], b0 = back[r], returned = back[r + 1] - b0, f0 = fresh[r];
  const int count = tail[0], have = tail[1];
  const int shift = s.shift ? s.shift[r] : 0;
  int32_t* table = s.tables + r * s.table_stride;
  for (int k = part * kFillThreads + tid; k < returned; k += parts * kFillThreads)
    if (count + b0 + k < have) s.free_list[count + b0 + k] = table[k];
  const Share mine = share_of(ask, give, t0, s.total, part, parts);
  const uint32_t i0 = mine.from, i1 = mine.to, rows = max(s.total - t0, 0);   // tokens i < rows have a row
  if (i0 >= i1) return;
  if (give == 0) {   // refused
    for (uint32_t i = i0 + tid; i < i1; i += kFillThreads) {
      s.out_slots[t0 + i] = -1;
      s.out_positions[t0 + i] = (long long)n + i + shift;
    }
    return;
  }
  // the blocks of these tokens, kFillBlocks at a time, then the tokens in them
  const uint32_t held = ((uint32_t)n + b - 1) / b, first = ((uint32_t)n + i0) / b, last = ((uint32_t)n + i1 - 1) / b;
  int row_lo = 0, row_hi = R - 1;   // the requests whose blocks came back and go to this one
  if (last >= held) {
    const int top = have - 1 - (f0 + (int)(max(first, held) - held)), low = have - 1 - (f0 + (int)(last - held));
    if (top >= count) {
      row_hi = warp_row_of(back, R, top - count);
      row_lo = warp_row_of(back, R, max(low - count, 0));
    }
  }
  for (uint32_t c = first; c <= last; c += kFillBlocks) {
    const int blocks = (int)min(last - c + 1, (uint32_t)kFillBlocks);
    __syncthreads();
    for (int k = tid; k < blocks; k += kFillThreads) {
      const uint32_t bi = c + k;
      int id;
      if (bi < held) {
        id = table[bi];
      } else {
        const int j = have - 1 - (f0 + (int)(bi - held));   // from the bottom of the stack, what came back on top
        if (j < count) {
          id = s.free_list[j];
        } else {
          int lo = row_lo, hi = row_hi;
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (back[mid] <= j - count) lo = mid;
            else hi = mid - 1;
          }
          id = s.tables[lo * s.table_stride + (j - count - back[lo])];
        }
        const int64_t at = (int64_t)bi * b - n;             // the block's first token: its part writes the entry
        if (at >= i0 && at < i1) table[bi] = id;
      }
      s_id[k] = id;
    }
    __syncthreads();
    const int64_t from = max((int64_t)i0, (int64_t)c * b - n), to = min((int64_t)i1, (int64_t)(c + blocks) * b - n);
    for (uint32_t i = (uint32_t)from + tid; i < to; i += kFillThreads) {
      const uint32_t pos = (uint32_t)n + i, bi = pos / b;
      if (i < rows) {
        s.out_slots[t0 + i] = (long long)s_id[bi - c] * b + (pos - bi * b);
        s.out_positions[t0 + i] = (long long)pos + shift;
      }
    }
  }
}

cudaError_t launch_block_tables(const ckv_table_step& s, cudaStream_t st) {
  const size_t smem = (size_t)(5 * s.requests + 3) * sizeof(int);
  if (cudaError_t e = ensure_dynamic_smem((const void*)k_block_tables, smem); e != cudaSuccess) return e;
  const bool solo = (int64_t)s.total + s.requests <= CKV_TABLES_SMALL;
  if (cudaError_t e = launch_after(k_block_tables, dim3(1), kTabThreads, smem, st, s, solo ? 1 : 0); solo || e != cudaSuccess)
    return e;
  // up to about four CTAs per SM, with work for each of their threads: a CTA costs more than it
  // saves without (16 requests, 23,000 tokens: 37 CTAs each 9.1 us, 12 each 7.2; 200 requests, 127,000
  // tokens: 2 each 8.8 us, 1 each 12, 11 each 13)
  const int most = s.requests >= 592 ? 1 : std::min(592 / s.requests, 64);
  const int parts = (int)std::min((int64_t)most, s.total / ((int64_t)kFillThreads * s.requests) + 1);
  return launch_after(k_block_tables_fill, dim3(s.requests + 1, parts), kFillThreads, 0, st, s);
}

}  // namespace ckv
