// Block tables, slots and positions of one decode / admission step, from the requests'
// lengths, on the device: a step of a captured graph can admit, extend and end requests
// without the host.
//
// With b tokens per block, request r holds ceil(len / b) blocks and needs
// ceil((len + new) / b) - ceil(len / b) more; new < 0 ends it and gives its blocks back.
// The free blocks are a stack.  Blocks given back go on top (requests in order, blocks in
// order); fresh blocks come off the top (requests in order, blocks in order).  All of it is
// three prefix sums over the requests (tokens, blocks back, blocks needed), held in shared
// memory by every CTA, after which each token and each block finds its request by binary
// search and is written independently.
//
// Bound: latency (a few loads per request, one dependent scan, one round of stores).  One
// CTA handles a decode step; above kOneCta tokens a cluster of 8 CTAs shares the stores
// (the cluster, because the new lengths may overwrite the old ones in place: every CTA has
// to have read them before any CTA writes).
#include <cooperative_groups.h>

#include "ckv_cache.h"
#include "ckv_common.cuh"

namespace cg = cooperative_groups;

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

__global__ void __launch_bounds__(kTabThreads) k_block_tables(const ckv_table_step s) {
  extern __shared__ int tab_smem[];
  __shared__ Sum3 scratch[32];
  __shared__ int s_taken;
  const int R = s.requests, b = s.block_size, tid = threadIdx.x;
  int* cu = tab_smem;             // [R + 1] tokens before request r, as asked for
  int* back = cu + R + 1;         // [R + 1] blocks given back before request r
  int* fresh = back + R + 1;      // [R + 1] fresh blocks wanted before request r
  int* len = fresh + R + 1;       // [R] old length
  int* ok = len + R;              // [R] 1: the request's tokens are granted
  if (tid == 0) s_taken = 0;
  const int count = min(max(__ldcg(s.free_count), 0), s.free_capacity);
  Sum3 run = {0, 0, 0};
  for (int base = 0; base < R; base += blockDim.x) {
    const int r = base + tid;
    Sum3 v = {0, 0, 0};
    if (r < R) {
      const int n = max(__ldcg(s.lens + r), 0), nw = __ldcg(s.new_tokens + r);
      const int held = (int)(((long long)n + b - 1) / b);
      len[r] = n;
      if (nw < 0) {
        v.back = min(held, s.table_width);
        ok[r] = 2;                // ended
      } else {
        v.tok = nw;
        const long long want = ((long long)n + nw + b - 1) / b;
        ok[r] = want <= s.table_width ? 1 : 0;
        v.need = ok[r] ? (int)want - held : 0;
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
    const int need = fresh[r + 1] - fresh[r];
    if (ok[r] == 1 && need > 0) {
      if (fresh[r + 1] <= have) atomicMax(&s_taken, fresh[r + 1]);
      else ok[r] = 0;
    }
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();   // every CTA has read the old lengths and the old count
  const int rank = (int)cl.block_rank(), nranks = (int)cl.num_blocks();
  const int gt = rank * blockDim.x + tid, gn = nranks * blockDim.x;
  const int taken = s_taken;

  // the j-th block from the bottom of the stack, after the blocks given back went on top
  auto stack = [&](int j) -> int {
    if (j < count) return __ldcg(s.free_list + j);
    const int e = j - count, r = row_of(back, 0, R - 1, e);
    return __ldcg(s.tables + r * s.table_stride + (e - back[r]));
  };
  for (int i = gt; i < have - count; i += gn) s.free_list[count + i] = stack(count + i);
  for (int i = gt; i < taken; i += gn) {
    const int r = row_of(fresh, 0, R - 1, i);
    s.tables[r * s.table_stride + (len[r] + b - 1) / b + (i - fresh[r])] = stack(have - 1 - i);
  }
  for (int r = gt; r <= R; r += gn) {
    s.out_cu[r] = cu[r];
    if (r == R) break;
    const int give = ok[r] == 1 ? cu[r + 1] - cu[r] : 0;
    s.out_granted[r] = give;
    s.out_lens[r] = ok[r] == 2 ? 0 : len[r] + give;
  }
  if (gt == 0) s.out_free_count[0] = have - taken;

  // tokens: a warp takes 128 at a time, its rows bracketed by two searches
  const int lane = tid & 31, asked = cu[R];
  for (int t0 = (gt >> 5) * 128; t0 < s.total; t0 += (gn >> 5) * 128) {
    const int first = row_of(cu, 0, R - 1, min(t0, max(asked - 1, 0)));
    const int last = row_of(cu, first, R - 1, min(t0 + 127, max(asked - 1, 0)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + i * 32 + lane;
      if (t >= s.total) break;
      long long slot = -1, where = 0;
      if (t < asked) {
        const int r = row_of(cu, first, last, t);
        const long long pos = (long long)len[r] + (t - cu[r]);
        where = pos + (s.shift ? s.shift[r] : 0);
        if (ok[r] == 1) {
          const int bi = (int)(pos / b), held = (len[r] + b - 1) / b;
          const int block = bi < held ? __ldcg(s.tables + r * s.table_stride + bi)
                                      : stack(have - 1 - (fresh[r] + bi - held));
          slot = (long long)block * b + pos % b;
        }
      }
      s.out_slots[t] = slot;
      s.out_positions[t] = where;
    }
  }
}

constexpr int kOneCta = 8192;   // tokens up to which one CTA makes the step

cudaError_t launch_block_tables(const ckv_table_step& s, cudaStream_t st) {
  const size_t smem = (size_t)(5 * s.requests + 3) * sizeof(int);
  if (cudaError_t e = ensure_dynamic_smem((const void*)k_block_tables, smem); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  const int ctas = s.total > kOneCta ? 8 : 1;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kTabThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_block_tables, s);
}

}  // namespace ckv
