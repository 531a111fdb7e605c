// Rotary positions of queries and keys, both in one launch.
//
// Pair i of a head turns by the angle position * f_i: (a, b) -> (a c - b s, b c + a s) with
// c, s = factor * cos, sin.  `inverse` turns by the negative angle, which is the transpose
// and so the gradient with respect to the unrotated vector.  The pairs are (x[i], x[i + d/2])
// or, interleaved, (x[2i], x[2i + 1]), for the first d dimensions; the rest pass through.
//
// Angles: position * f / 2 pi in 64 bits, reduced to a fraction of a turn in (-1/2, 1/2],
// then single precision with the residual of that rounding put back to first order, so a
// position of 10^6 loses nothing (in 32 bits its angle would be off by 0.06).  They are
// computed once per token and shared by all heads through shared memory.
//
// Bound: HBM (each element read once and written once): 32768 tokens of 40 heads of 128 in bf16 104 us
// (the kernel alone), 6.5 TB/s; 8191 in fp32 with 64 of 128 dimensions interleaved 58 us, 5.8 TB/s.
#include <algorithm>

#include "ckv_cache.h"
#include "ckv_common.cuh"

namespace ckv {

constexpr int kRotThreads = 256;

template <typename T> CKV_DEV T from_f32(float x);
template <> CKV_DEV float from_f32<float>(float x) { return x; }
template <> CKV_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> CKV_DEV __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T x[N]; };

// Cosine and sine (times factor) of tokens t0 .. t0 + nt, [nt][pairs] in shared memory.
CKV_DEV void turns_of(const ckv_rotary_args& a, int t0, int nt, float2* cs) {
  after_previous();
  const int pairs = a.rotary_dim / 2;
  for (int i = threadIdx.x; i < nt * pairs; i += kRotThreads) {
    const int t = i / pairs, p = i - t * pairs;
    const double turns = (double)a.positions[t0 + t] * (a.inv_freq[p] * 0.15915494309189533577);
    const double r = turns - rint(turns);
    const float hi = (float)r, lo = (float)(r - (double)hi) * 6.2831853f;
    float s, c;
    sincospif(2.f * hi, &s, &c);
    const float c1 = fmaf(-lo, s, c), s1 = fmaf(lo, c, s);
    cs[i] = make_float2(c1 * a.factor, (a.inverse ? -s1 : s1) * a.factor);
  }
  __syncthreads();
}

// A unit is 2N elements: N of the first half and their N partners (half layout), or 2N adjacent
// ones (interleaved), or 2N past the rotated part (N at its end, where that is odd).
template <typename T, int N, bool kInter>
__global__ void __launch_bounds__(kRotThreads) k_rotary(const ckv_rotary_args a, int tokens_per_cta) {
  extern __shared__ float2 rot_cs[];   // [tokens_per_cta][pairs]
  const int t0 = blockIdx.x * tokens_per_cta;
  const int pairs = a.rotary_dim / 2, nt = min(tokens_per_cta, a.tokens - t0);
  turns_of(a, t0, nt, rot_cs);
  const int turn_units = pairs / N;                                   // per head
  const int rest_units = (a.head_dim - a.rotary_dim + 2 * N - 1) / (2 * N);
  const int units = turn_units + rest_units;
  const int heads = a.q_heads + a.k_heads;
  const int h0 = blockIdx.y * a.heads_per_cta, h1 = min(heads, h0 + a.heads_per_cta);
  const int per_token = (h1 - h0) * units;
  for (int i = threadIdx.x; i < nt * per_token; i += kRotThreads) {
    const int t = i / per_token, j = i - t * per_token;
    const int hh = j / units, u = j - hh * units;
    const int h = h0 + hh;
    const bool isk = h >= a.q_heads;
    const int64_t tok = t0 + t;
    const T* src = isk ? static_cast<const T*>(a.k) + tok * a.k_tok_stride + (h - a.q_heads) * a.k_head_stride
                       : static_cast<const T*>(a.q) + tok * a.q_tok_stride + h * a.q_head_stride;
    T* dst = isk ? static_cast<T*>(a.out_k) + tok * a.out_k_tok_stride + (h - a.q_heads) * a.out_k_head_stride
                 : static_cast<T*>(a.out_q) + tok * a.out_q_tok_stride + h * a.out_q_head_stride;
    using V = Vec<T, N>;
    if (u < turn_units) {
      const float2* cs = rot_cs + t * pairs + u * N;
      const int i0 = kInter ? 2 * u * N : u * N, i1 = kInter ? i0 + N : i0 + pairs;
      const V x = *reinterpret_cast<const V*>(src + i0), y = *reinterpret_cast<const V*>(src + i1);
      V ox, oy;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (!kInter) {
          const float c = cs[e].x, s = cs[e].y, p = to_f32(x.x[e]), q = to_f32(y.x[e]);
          ox.x[e] = from_f32<T>(p * c - q * s);
          oy.x[e] = from_f32<T>(q * c + p * s);
        } else if (e % 2 == 0) {
          const float c = cs[e / 2].x, s = cs[e / 2].y, p = to_f32(x.x[e]), q = to_f32(x.x[e + 1]);
          ox.x[e] = from_f32<T>(p * c - q * s);
          ox.x[e + 1] = from_f32<T>(q * c + p * s);
          const float c2 = cs[N / 2 + e / 2].x, s2 = cs[N / 2 + e / 2].y;
          const float p2 = to_f32(y.x[e]), q2 = to_f32(y.x[e + 1]);
          oy.x[e] = from_f32<T>(p2 * c2 - q2 * s2);
          oy.x[e + 1] = from_f32<T>(q2 * c2 + p2 * s2);
        }
      }
      *reinterpret_cast<V*>(dst + i0) = ox;
      *reinterpret_cast<V*>(dst + i1) = oy;
    } else if (src != dst) {
      const int i0 = a.rotary_dim + (u - turn_units) * 2 * N, i1 = i0 + N;
      const V x = *reinterpret_cast<const V*>(src + i0);
      if (i1 < a.head_dim) *reinterpret_cast<V*>(dst + i1) = *reinterpret_cast<const V*>(src + i1);
      *reinterpret_cast<V*>(dst + i0) = x;
    }
  }
}

// Any rotary dimension, element by element: a warp has a row (token, head) and its lanes the pairs.
// kStaged: 16-bit rows that start on 16 bytes go through shared memory, read and written in 16-byte
// pieces, a few rows at a time; otherwise any alignment.  (8192 tokens of 40 heads, 122 of 128
// dimensions in bf16: 112 us as units of the kernel above with N = 1, 90 by rows, 82 staged; fp32, 58 of
// 64: 60, 55, 65.)
template <typename T, bool kInter, bool kStaged>
__global__ void __launch_bounds__(kRotThreads) k_rotary_rows(const ckv_rotary_args a, int tokens_per_cta, int batch) {
  extern __shared__ float2 rot_cs[];
  const int t0 = blockIdx.x * tokens_per_cta;
  const int pairs = a.rotary_dim / 2, nt = min(tokens_per_cta, a.tokens - t0);
  turns_of(a, t0, nt, rot_cs);
  const int h0 = blockIdx.y * a.heads_per_cta, nh = min(a.q_heads + a.k_heads - h0, a.heads_per_cta);
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  auto home = [&](int row, const T*& src, T*& dst) {
    const int t = row / nh, h = h0 + row - t * nh;
    const int64_t tok = t0 + t;
    if (h >= a.q_heads) {
      src = static_cast<const T*>(a.k) + tok * a.k_tok_stride + (h - a.q_heads) * a.k_head_stride;
      dst = static_cast<T*>(a.out_k) + tok * a.out_k_tok_stride + (h - a.q_heads) * a.out_k_head_stride;
    } else {
      src = static_cast<const T*>(a.q) + tok * a.q_tok_stride + h * a.q_head_stride;
      dst = static_cast<T*>(a.out_q) + tok * a.out_q_tok_stride + h * a.out_q_head_stride;
    }
  };
  auto turn = [&](const T* src, T* dst, const float2* cs) {
#pragma unroll 2
    for (int p = lane; p < pairs; p += 32) {
      const int i0 = kInter ? 2 * p : p, i1 = kInter ? i0 + 1 : p + pairs;
      const float x = to_f32(src[i0]), y = to_f32(src[i1]);
      dst[i0] = from_f32<T>(x * cs[p].x - y * cs[p].y);
      dst[i1] = from_f32<T>(y * cs[p].x + x * cs[p].y);
    }
  };
  const T* src;
  T* dst;
  if constexpr (kStaged) {
    const int vecs = a.head_dim * (int)sizeof(T) / 16;   // of a row
    uint4* stage = reinterpret_cast<uint4*>(rot_cs + ((tokens_per_cta * pairs + 1) & ~1)) + wid * batch * vecs;
    for (int row0 = wid * batch; row0 < nt * nh; row0 += kRotThreads / 32 * batch) {
      const int rows = min(batch, nt * nh - row0);
      for (int v = lane; v < rows * vecs; v += 32) {
        const int r = v / vecs;
        home(row0 + r, src, dst);
        stage[v] = reinterpret_cast<const uint4*>(src)[v - r * vecs];
      }
      __syncwarp();
      for (int r = 0; r < rows; ++r) {
        T* x = reinterpret_cast<T*>(stage + r * vecs);
        turn(x, x, rot_cs + (row0 + r) / nh * pairs);
      }
      __syncwarp();
      for (int v = lane; v < rows * vecs; v += 32) {
        const int r = v / vecs;
        home(row0 + r, src, dst);
        reinterpret_cast<uint4*>(dst)[v - r * vecs] = stage[v];
      }
      __syncwarp();
    }
  } else {
    for (int row = wid; row < nt * nh; row += kRotThreads / 32) {
      home(row, src, dst);
      turn(src, dst, rot_cs + row / nh * pairs);
      if (src != dst)
        for (int d = a.rotary_dim + lane; d < a.head_dim; d += 32) dst[d] = src[d];
    }
  }
}

template <typename T, int N>
static cudaError_t rot_launch(const ckv_rotary_args& a, int tpc, dim3 grid, bool rows16, cudaStream_t st) {
  const size_t table = ((size_t)tpc * (a.rotary_dim / 2) + 1) / 2 * 2 * sizeof(float2);
  if constexpr (N > 1) {
    return launch_after(a.interleaved ? k_rotary<T, N, true> : k_rotary<T, N, false>, grid, kRotThreads, table, st, a, tpc);
  } else if (rows16 && sizeof(T) == 2) {
    const int row = a.head_dim * (int)sizeof(T), batch = std::max(1, 1024 / row);   // 1 KB per warp in flight
    const size_t smem = table + (size_t)(kRotThreads / 32) * batch * row;
    auto fn = a.interleaved ? k_rotary_rows<T, true, true> : k_rotary_rows<T, false, true>;
    if (cudaError_t e = ensure_dynamic_smem((const void*)fn, smem); e != cudaSuccess) return e;
    return launch_after(fn, grid, kRotThreads, smem, st, a, tpc, batch);
  } else {
    return launch_after(a.interleaved ? k_rotary_rows<T, true, false> : k_rotary_rows<T, false, false>, grid, kRotThreads, table, st,
                        a, tpc, 1);
  }
}

cudaError_t launch_rotary(const ckv_rotary_args& args, cudaStream_t st) {
  ckv_rotary_args a = args;
  const int es = a.dtype == CKV_FP32 ? 4 : 2, n = 16 / es;
  const int heads = a.q_heads + a.k_heads;
  // 16-byte vectors need every row and every half to start on 16 bytes
  auto al = [&](const void* p, int64_t ts, int64_t hs) {
    return (uintptr_t)p % 16 == 0 && (ts * es) % 16 == 0 && (hs * es) % 16 == 0;
  };
  const bool rows16 = al(a.q, a.q_tok_stride, a.q_head_stride) && al(a.out_q, a.out_q_tok_stride, a.out_q_head_stride) &&
                   (a.k_heads == 0 || (al(a.k, a.k_tok_stride, a.k_head_stride) &&
                                       al(a.out_k, a.out_k_tok_stride, a.out_k_head_stride))) &&
                      a.head_dim % n == 0;
  const bool vec = rows16 && (a.rotary_dim / 2) % n == 0;
  // few tokens: one per CTA and the heads spread over CTAs (latency); many: four per CTA share the angles'
  // barrier.  40 heads of 128 in bf16, kernel alone: 16 tokens in 8 splits 1.9 us, in 1 2.3, four per CTA
  // 4.0; 148 in 2 splits 2.1, in 8 2.7; 1024 in 2 splits 6.0, four per CTA 9.8; 4096: 16.4 and 17.1; 8192:
  // one per CTA 33, four 30; 32768: 117 and 104
  const int tpc = a.tokens >= 1024 ? 4 : 1;
  const int splits = a.tokens >= 1024 ? 1 : (a.tokens >= 148 ? 2 : 8);
  a.heads_per_cta = (heads + splits - 1) / splits;
  const dim3 grid((a.tokens + tpc - 1) / tpc, (heads + a.heads_per_cta - 1) / a.heads_per_cta);
  switch (a.dtype) {
    case CKV_BF16: return vec ? rot_launch<__nv_bfloat16, 8>(a, tpc, grid, rows16, st) : rot_launch<__nv_bfloat16, 1>(a, tpc, grid, rows16, st);
    case CKV_FP16: return vec ? rot_launch<__half, 8>(a, tpc, grid, rows16, st) : rot_launch<__half, 1>(a, tpc, grid, rows16, st);
    default: return vec ? rot_launch<float, 4>(a, tpc, grid, rows16, st) : rot_launch<float, 1>(a, tpc, grid, rows16, st);
  }
}

}  // namespace ckv
