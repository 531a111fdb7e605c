// Write and read of the paged 8-bit decode cache.
//
// Keys and values are held in 8 bits (e4m3 or int8) with one scale for each (block, KV
// head): the smallest power of two, 2^-126 at least, with max |x| / scale at most the
// format's largest value (448, 127).  Powers of two make x / scale exact, so a code is
// the one rounding of its value, and when a later token raises a block's scale the e4m3
// codes move by an exponent without a second rounding (above the subnormals); int8 codes are
// shifted and rounded once.  A NaN or an infinity makes the scale NaN: everything read from
// that (block, head) is NaN rather than quietly wrong.
//
// Write.  The call's tokens come with their slots; neighbours in one block form a run.  A CTA
// owns the runs that begin in its piece of the token list, for one head and one of K / V: all
// warps read the run's rows once into registers (16 rows per warp), the CTA agrees on the
// largest magnitude, the block's scale follows, and the rows leave as codes.  A run that has
// the block's first token begins the block anew; any other run keeps what the block holds,
// rescaled when the scale grew, or when another program left one that is no power of two (the next
// one takes its place).  One CTA per (run, head, K / V), so no atomics and the same
// result every time.
//
// Bound: HBM, (element size + 1) bytes per element, and the latency of a run's chain: 16 prompts of
// 33,421 tokens, 8 heads of 128 in bf16: 37 us, 4.6 TB/s.  Reading (k_cache_read) has no such chain:
// 131,072 tokens written and read, fp16, int8: 263 us, 6.1 TB/s.
#include <type_traits>

#include "ckv_cache.h"
#include "ckv_common.cuh"

namespace ckv {

constexpr int kRowsPerWarp = 16;

// Smallest power-of-two scale (as a float) for a largest magnitude given by its bits; NaN for
// a NaN or an infinity.  448 = 1.75 2^8, 127 = 1.984375 2^6.
template <int kFmt> CKV_DEV float scale_for(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  constexpr uint32_t kMant = kFmt == CKV_CACHE_E4M3 ? 0x600000u : 0x7e0000u;
  constexpr int kExp = kFmt == CKV_CACHE_E4M3 ? 8 : 6;
  int e = (int)(amax_bits >> 23) - kExp + ((amax_bits & 0x7fffffu) > kMant ? 1 : 0);   // biased by 127
  e = max(e, 1);   // 2^-126, also for zero and subnormal magnitudes
  return __uint_as_float((uint32_t)e << 23);
}
// 1 / scale of a power of two in [2^-126, 2^127] (a subnormal of the last).
CKV_DEV float inv_pow2(float s) { return __uint_as_float(max((254u << 23) - __float_as_uint(s), 0x400000u)); }
// The smallest power of two that is at least a positive s; infinity above 2^127.
CKV_DEV float up_pow2(float s) { return __uint_as_float((__float_as_uint(s) + 0x7fffffu) & 0x7f800000u); }

// Four codes from four values over the scale, or (by) codes of another scale times its ratio to it.
// int8: adding 1.5 2^23 leaves the nearest whole number, ties to even, in the low byte; with the
// multiplication in one instruction, so that the product is not rounded first.
template <int kFmt> CKV_DEV uint32_t encode4(float a, float b, float c, float d, float by = 1.f) {
  uint32_t r;
  if constexpr (kFmt == CKV_CACHE_E4M3) {
    asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
        "mov.b32 %0, {lo, hi};\n}\n" : "=r"(r) : "f"(a * by), "f"(b * by), "f"(c * by), "f"(d * by));
  } else {
    constexpr float kMagic = 12582912.f;
    const uint32_t x = __float_as_uint(fmaf(a, by, kMagic)), y = __float_as_uint(fmaf(b, by, kMagic));
    const uint32_t z = __float_as_uint(fmaf(c, by, kMagic)), w = __float_as_uint(fmaf(d, by, kMagic));
    r = __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  }
  return r;
}
template <int kFmt> CKV_DEV void decode4(uint32_t w, float (&o)[4]) {
  if constexpr (kFmt == CKV_CACHE_E4M3) {
    uint32_t lo, hi;
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 p = __half22float2(*reinterpret_cast<__half2*>(&lo)), q = __half22float2(*reinterpret_cast<__half2*>(&hi));
    o[0] = p.x; o[1] = p.y; o[2] = q.x; o[3] = q.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (float)(int8_t)(w >> (8 * i));
  }
}

// 16 elements of a row as they are, their largest magnitude, and four of them as fp32 times a
// power of two.
template <typename T> struct Row16;
template <> struct Row16<float> {
  float4 x[4];
  CKV_DEV void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = reinterpret_cast<const float4*>(p)[i];
  }
  CKV_DEV void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  CKV_DEV float4 get(int i, float by) const { return make_float4(x[i].x * by, x[i].y * by, x[i].z * by, x[i].w * by); }
  CKV_DEV uint32_t amax(uint32_t top) const {   // a NaN stays
    float m = __uint_as_float(top);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m = max3_abs(m, x[i].x, x[i].y);
      m = max3_abs(m, x[i].z, x[i].w);
    }
    return __float_as_uint(m);
  }
  static CKV_DEV float max3_abs(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
  }
  static CKV_DEV uint32_t fp32_bits(uint32_t top) { return top & 0x7fffffffu; }
};
template <typename H> struct Row16 {
  uint32_t w[8];
  CKV_DEV void load(const H* p) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
  CKV_DEV void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
  }
  CKV_DEV float4 get(int i, float by) const {
    if constexpr (std::is_same<H, __half>::value) {   // `by` may be out of its range
      const float2 a = f2(w[2 * i]), b = f2(w[2 * i + 1]);
      return make_float4(a.x * by, a.y * by, b.x * by, b.y * by);
    } else {   // exact in bf16 too, above 2^-126 (every format's zero)
      const uint32_t by2 = __byte_perm(__float_as_uint(by), 0, 0x3232);
      uint32_t x, y;
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(w[2 * i]), "r"(by2));
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(w[2 * i + 1]), "r"(by2));
      const float2 a = f2(x), b = f2(y);
      return make_float4(a.x, a.y, b.x, b.y);
    }
  }
  CKV_DEV uint32_t amax(uint32_t top) const {   // of both halves of the words, of any sign; a NaN stays
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same<H, __half>::value) asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(top) : "r"(w[i]));
      else asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(w[i]));
    }
    return top;
  }
  static CKV_DEV uint32_t fp32_bits(uint32_t top) {   // ordered as the magnitudes, a NaN on top
    const float2 m = f2(top & 0x7fff7fffu);
    return max(__float_as_uint(m.x), __float_as_uint(m.y));
  }
  static CKV_DEV float2 f2(uint32_t v) {
    if constexpr (sizeof(H) == 2 && std::is_same<H, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  }
};
CKV_DEV void store16(float* p, const float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}
CKV_DEV uint32_t pack2(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
CKV_DEV uint32_t pack2(float a, float b, __half*) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename H> CKV_DEV void store16(H* p, const float (&x)[16]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack2(x[2 * i], x[2 * i + 1], (H*)nullptr);
  reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

struct WriteArgs {
  ckv_cache c;
  CacheRows r;
  int piece;       // tokens of the list whose runs a CTA owns
  int block_log2;
  int items;       // of the 2 * heads (head, K / V) pairs, how many a CTA writes
};

constexpr int kSlotWindow = 2 * kCacheMaxBlock + 2;

// grid (pieces, 2 * heads / items); block_size / 16 warps.
template <typename T, int kFmt, int D>
__global__ void __launch_bounds__(kCacheMaxBlock / kRowsPerWarp * 32) k_cache_write(const WriteArgs a) {
  constexpr int kLanesPerRow = D / 16, kRowsPerStep = 32 / kLanesPerRow, kSteps = kRowsPerWarp / kRowsPerStep;
  __shared__ uint32_t s_max[2][kCacheMaxBlock / kRowsPerWarp];   // of this item and the next
  __shared__ uint32_t s_new[kCacheMaxBlock / 32];                // places of the block that this run writes
  __shared__ int s_slot[2][kSlotWindow];                          // block (-1: none) and place of the tokens from T0 - 1 on
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int bs = a.c.block_size, T0 = blockIdx.x * a.piece, T1 = min(a.r.tokens, T0 + a.piece);
  const int item0 = blockIdx.y * a.items, item1 = min(2 * a.c.num_kv_heads, item0 + a.items);
  const int64_t pool = (int64_t)a.c.num_blocks << a.block_log2;
  const int64_t* slots = a.r.slots;
  auto decode = [&](int i, int& blk, int& place) {
    const int64_t s = i >= 0 && i < a.r.tokens ? slots[i] : -1;
    blk = s >= 0 && s < pool ? (int)(s >> a.block_log2) : -1;
    place = (int)s & (bs - 1);
  };
  after_previous();
  // the piece's slots and those that a run may reach, in one reading
  const int window = T1 - T0 + bs + 2;
  for (int j = threadIdx.x; j < window; j += blockDim.x) decode(T0 - 1 + j, s_slot[0][j], s_slot[1][j]);
  __syncthreads();
  auto block_of = [&](int i) -> int {
    if (i - T0 + 1 < window) return s_slot[0][i - T0 + 1];
    int blk, place;
    decode(i, blk, place);
    return blk;
  };
  auto place_at = [&](int i) -> int {
    if (i - T0 + 1 < window) return s_slot[1][i - T0 + 1];
    int blk, place;
    decode(i, blk, place);
    return place;
  };
  int t = T0;
  while (t < T1) {   // every warp takes the same path
    // the next token that begins a run: its block is not the token's before it
    const int cand = t + lane;
    const int mine = cand < T1 ? block_of(cand) : -1;
    const uint32_t begins = __ballot_sync(0xffffffffu, mine >= 0 && block_of(cand - 1) != mine);
    if (begins == 0) { t += 32; continue; }
    t += __ffs(begins) - 1;
    const int blk = __shfl_sync(0xffffffffu, mine, __ffs(begins) - 1);
    // the run's end, and whether it has the block's first token and rising places
    int end = t;
    bool rising = true, anew = false;
    for (bool more = true; more;) {
      const int i = end + lane;
      const uint32_t m = __ballot_sync(0xffffffffu, block_of(i) == blk);
      const int n = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
      const bool own = lane < n;
      const int place = own ? place_at(i) : -1;
      rising = rising && __all_sync(0xffffffffu, !own || i == t || place_at(i - 1) < place);
      anew = anew || __any_sync(0xffffffffu, place == 0);
      end += n;
      more = n == 32;
    }
    if (!anew) {
      if (threadIdx.x < kCacheMaxBlock / 32) s_new[threadIdx.x] = 0;
      __syncthreads();
      for (int i = t + threadIdx.x; i < end; i += blockDim.x) {
        const int o = place_at(i);
        atomicOr(&s_new[o >> 5], 1u << (o & 31));
      }
    }
    // the rows of this thread in the first round (a longer run names slots twice)
    const int rows_per_round = nw * kRowsPerWarp;
    const bool once = end - t <= rows_per_round;
    const int row0 = t + wid * kRowsPerWarp + lane / kLanesPerRow, col = (lane % kLanesPerRow) * 16;
    // where row i goes; -1: past the run, or its slot is named again later (its last token stays)
    auto place_of = [&](int i) -> int {
      if (i >= end) return -1;
      const int o = place_at(i);
      if (!rising)
        for (int j = i + 1; j < end; ++j)
          if (place_at(j) == o) return -1;
      return o;
    };
    int place[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) place[s] = place_of(row0 + s * kRowsPerStep);
#pragma unroll 1
    for (int item = item0; item < item1; ++item) {
      const int h = item >> 1;
      const bool isv = item & 1;
      const T* src = static_cast<const T*>(isv ? a.r.v : a.r.k) + h * (isv ? a.r.vhs : a.r.khs) + col;
      const int64_t ts = isv ? a.r.vts : a.r.kts;
      char* dst = static_cast<char*>(isv ? a.c.v : a.c.k) + blk * (isv ? a.c.v_block_stride : a.c.k_block_stride) +
                  h * (isv ? a.c.v_head_stride : a.c.k_head_stride) + col;
      const int64_t tstr = isv ? a.c.v_tok_stride : a.c.k_tok_stride;
      float* at = (isv ? a.c.v_scale : a.c.k_scale) + (int64_t)blk * a.c.num_kv_heads + h;
      const float old = anew ? 0.f : *at;
      Row16<T> x[kSteps];
      uint32_t top = 0;
#pragma unroll 1
      for (int r0 = row0; r0 - row0 < end - t; r0 += rows_per_round) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int i = r0 + s * kRowsPerStep;
          if (i < end) x[s].load(src + i * ts);
          else x[s].clear();
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) top = x[s].amax(top);
      }
      top = __reduce_max_sync(0xffffffffu, Row16<T>::fp32_bits(top));
      if (nw > 1 || !anew) {
        uint32_t* all = s_max[item & 1];
        if (lane == 0) all[wid] = top;
        __syncthreads();   // s_new is whole, and every warp has read the item's old scale
        for (int w = 0; w < nw; ++w) top = max(top, all[w]);
      }
      float scale = scale_for<kFmt>(top);
      if (isnan(old) || isnan(scale) || isinf(up_pow2(old))) scale = __uint_as_float(0x7fffffffu);
      else scale = fmaxf(scale, up_pow2(old));
      const bool bad = isnan(scale);
      const float inv = bad ? 0.f : inv_pow2(scale);
      auto put = [&](const Row16<T>& row, int o) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 f = row.get(e, inv);
          w[e] = encode4<kFmt>(f.x, f.y, f.z, f.w);
        }
        if (bad) w[0] = w[1] = w[2] = w[3] = 0;
        *reinterpret_cast<uint4*>(dst + o * tstr) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      if (once) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          if (place[s] >= 0) put(x[s], place[s]);
      } else {
        for (int r0 = row0; r0 - row0 < end - t; r0 += rows_per_round)
#pragma unroll 1
          for (int s = 0; s < kSteps; ++s) {
            const int i = r0 + s * kRowsPerStep, o = place_of(i);
            if (o < 0) continue;
            x[0].load(src + i * ts);
            put(x[0], o);
          }
      }
      if (!anew && !bad && scale > old) {   // the tokens that stay, in the new scale
        const float ratio = old * inv;
#pragma unroll 1
        for (int s = 0; s < kSteps; ++s) {
          const int o = wid * kRowsPerWarp + s * kRowsPerStep + lane / kLanesPerRow;
          if (s_new[o >> 5] >> (o & 31) & 1u) continue;
          uint4* p = reinterpret_cast<uint4*>(dst + o * tstr);
          const uint4 v = *p;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f[4];
            decode4<kFmt>(w[e], f);
            w[e] = encode4<kFmt>(f[0], f[1], f[2], f[3], ratio);
          }
          *p = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      if (threadIdx.x == 0) *at = scale;
    }
    t = end;
    __syncthreads();   // s_new and s_max are free for the next run
  }
}

// A thread has 16 codes of K and of V of kReadTokens tokens (two of them half the list apart):
// the slots first, then all codes and scales, then the stores, so that four loads of 16 bytes
// are in flight.
constexpr int kReadTokens = 2;
template <typename T, int kFmt>
__global__ void __launch_bounds__(256) k_cache_read(const ckv_cache c, const CacheRows r, int block_log2) {
  const uint32_t per_row = c.head_dim / 16, per_tok = per_row * c.num_kv_heads;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, half = (r.tokens + kReadTokens - 1) / kReadTokens;
  const uint32_t t = i / per_tok;
  after_previous();
  if (t >= half) return;
  const uint32_t h = (i - t * per_tok) / per_row, v16 = i - t * per_tok - h * per_row;
  const int64_t pool = (int64_t)c.num_blocks << block_log2;
  int64_t slot[kReadTokens];
#pragma unroll
  for (int j = 0; j < kReadTokens; ++j) slot[j] = t + j * half < (uint32_t)r.tokens ? r.slots[t + j * half] : -1;
  uint4 q[kReadTokens][2];
  float sc[kReadTokens][2];
#pragma unroll
  for (int j = 0; j < kReadTokens; ++j)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      q[j][v] = make_uint4(0, 0, 0, 0);
      sc[j][v] = 0.f;
      if (slot[j] < 0 || slot[j] >= pool) continue;
      const int64_t blk = slot[j] >> block_log2, o = slot[j] & (c.block_size - 1);
      const char* p = v ? static_cast<const char*>(c.v) + blk * c.v_block_stride + h * c.v_head_stride + o * c.v_tok_stride
                        : static_cast<const char*>(c.k) + blk * c.k_block_stride + h * c.k_head_stride + o * c.k_tok_stride;
      q[j][v] = *(reinterpret_cast<const uint4*>(p) + v16);
      sc[j][v] = (v ? c.v_scale : c.k_scale)[blk * c.num_kv_heads + h];
    }
#pragma unroll
  for (int j = 0; j < kReadTokens; ++j)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (t + j * half >= (uint32_t)r.tokens) continue;
      const uint32_t w[4] = {q[j][v].x, q[j][v].y, q[j][v].z, q[j][v].w};
      float x[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
        decode4<kFmt>(w[e], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[4 * e + k] = f[k] * sc[j][v];
      }
      T* out = v ? static_cast<T*>(r.v) + (int64_t)(t + j * half) * r.vts + h * r.vhs
                 : static_cast<T*>(r.k) + (int64_t)(t + j * half) * r.kts + h * r.khs;
      store16(out + v16 * 16, x);
    }
}

static int log2_of(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}

template <typename T, int kFmt>
static cudaError_t write_launch(const WriteArgs& a, dim3 grid, int threads, cudaStream_t st) {
  return launch_after(a.c.head_dim == 64 ? k_cache_write<T, kFmt, 64> : k_cache_write<T, kFmt, 128>, grid, threads, 0, st, a);
}

cudaError_t launch_cache_write(const ckv_cache& c, const CacheRows& r, cudaStream_t st) {
  WriteArgs a;
  a.c = c; a.r = r; a.block_log2 = log2_of(c.block_size);
  // a decode step has a run per token: a CTA for each and each (head, K / V).  A prompt's runs are
  // whole blocks; a CTA that writes more pairs finds its run once for all of them, but fewer CTAs
  // hide less latency (131072 tokens of 8 heads: 2 pairs 137 us, 4 pairs 132; 33,000 tokens: 37, 39).
  // Up to 1024 tokens the host cannot tell one from the other: 256 appends to blocks of 32 take 7 us with a CTA
  // each and 61 in pieces, 1024 22 and 63 (8192: 165 and 126); one prompt of 256 tokens 5.3 and 3.8, of 1024 18 and 4.2
  a.piece = r.tokens <= 1024 ? 1 : c.block_size;
  const int pieces = (r.tokens + a.piece - 1) / a.piece, pairs = 2 * c.num_kv_heads;
  a.items = r.tokens <= 1024 ? 1 : (int64_t)pieces * pairs / 4 >= 148 * 32 ? 4 : 2;
  const dim3 grid(pieces, (pairs + a.items - 1) / a.items);
  const int threads = c.block_size / kRowsPerWarp * 32;
  const bool e4 = c.format == CKV_CACHE_E4M3;
  switch (r.dtype) {
    case CKV_BF16:
      return e4 ? write_launch<__nv_bfloat16, CKV_CACHE_E4M3>(a, grid, threads, st)
                : write_launch<__nv_bfloat16, CKV_CACHE_INT8>(a, grid, threads, st);
    case CKV_FP16:
      return e4 ? write_launch<__half, CKV_CACHE_E4M3>(a, grid, threads, st) : write_launch<__half, CKV_CACHE_INT8>(a, grid, threads, st);
    default:
      return e4 ? write_launch<float, CKV_CACHE_E4M3>(a, grid, threads, st) : write_launch<float, CKV_CACHE_INT8>(a, grid, threads, st);
  }
}

cudaError_t launch_cache_read(const ckv_cache& c, const CacheRows& r, cudaStream_t st) {
  const int64_t n = ((int64_t)r.tokens + kReadTokens - 1) / kReadTokens * c.num_kv_heads * (c.head_dim / 16);
  const dim3 grid((unsigned)((n + 255) / 256));
  const int bl = log2_of(c.block_size);
  const bool e4 = c.format == CKV_CACHE_E4M3;
  switch (r.dtype) {
    case CKV_BF16:
      return launch_after(e4 ? k_cache_read<__nv_bfloat16, CKV_CACHE_E4M3> : k_cache_read<__nv_bfloat16, CKV_CACHE_INT8>, grid, 256, 0,
                          st, c, r, bl);
    case CKV_FP16:
      return launch_after(e4 ? k_cache_read<__half, CKV_CACHE_E4M3> : k_cache_read<__half, CKV_CACHE_INT8>, grid, 256, 0, st, c, r, bl);
    default:
      return launch_after(e4 ? k_cache_read<float, CKV_CACHE_E4M3> : k_cache_read<float, CKV_CACHE_INT8>, grid, 256, 0, st, c, r, bl);
  }
}

}  // namespace ckv
