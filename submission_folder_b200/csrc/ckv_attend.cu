// Attention of a few query tokens per sequence over the paged 8-bit decode cache.
//
// out = sum_j softmax_j(scale q.k_j) v_j with k_j = ks[b] * ck_j, v_j = vs[b] * cv_j: codes
// c in 8 bits, scales by (block b, KV head).  One pass, with a running maximum.  The scales
// never touch the codes: ks multiplies the logit after its dot product, and vs joins the
// weight as an exponent, w_j = 2^(s_j + log2 vs - m'), which has its own running maximum m'
// beside the softmax's m; the two meet once, at the end.  So the matrix products run on the
// codes, which fp16 holds exactly.
//
// Precision: fp16 products with fp32 sums.  The other operands are split in two fp16 terms,
// x = hi + lo / 4096 (22 bits): the query rows after a power of two brings each row to
// [1, 2), and the weights, which lie in [0, 1].  The two terms fill rows 0-7 and 8-15 of one
// m16n8k16 product, whose 16 rows the few rows of a KV head (its query heads times the new
// tokens) leave half empty anyway, so the second term costs nothing.  The products of one
// step are summed by the tensor core and added to the output in fp32 with rounding (the
// tensor core truncates, which over thousands of steps would lean one way).
//
// Split: the unit of work is 32 tokens of one (sequence, KV head, tile of query rows).  All
// units stand in one line, which is cut evenly into one piece per CTA and then per warp, so a
// ragged batch, a single long sequence and a large batch fill the GPU alike, from lengths
// that only the device knows.  Each warp runs on its own: it copies its tokens' codes with
// cp.async into its own ring of shared memory (kStages - 1 steps ahead) and multiplies from
// there.  Pieces of one unit are merged in the CTA, then across CTAs by k_attend_merge in
// ascending order: no atomics, and the same bits every time.
//
// Bound: HBM (each code is read once).
#include "ckv_cache.h"
#include "ckv_common.cuh"

namespace ckv {

constexpr int kAttWarps = 8;
constexpr int kAttStep = 32;     // tokens per step
constexpr int kAttStages = 3;
constexpr int kAttMaxCtas = 148;

struct AttArgs {
  ckv_cache c;
  ckv_attention_args a;
  float* ws;                     // [ctas][kAttWarps + 2] partial results
  int4* desc;                    // [ctas][2]: what k_attend_merge has to merge from this CTA on
  int block_log2, group, ctas;
};

// A partial result: 8 * NT rows of (m, m', l, -) then of D sums.
__host__ __device__ constexpr int part_floats(int D, int rows) { return rows * (D + 4); }

// ---- small pieces -------------------------------------------------------------------
CKV_DEV uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
CKV_DEV void cp16(uint32_t dst, const void* src, uint32_t bytes) {   // bytes 0: zero fill, src not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
CKV_DEV void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
CKV_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> CKV_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
CKV_DEV uint4 lds4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
CKV_DEV uint2 lds2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
CKV_DEV float lds1(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
CKV_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four codes to two fp16 pairs, exactly.
template <int kFmt> CKV_DEV void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kFmt == CKV_CACHE_E4M3) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {   // 0x6400 | (code + 128) is the fp16 number 1024 + code + 128
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t k = 0x64806480u;
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&k));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&k));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
// (x, y) as two fp16 pairs: x ~ hi + lo / 4096.
CKV_DEV void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn((x - f.x) * 4096.f, (y - f.y) * 4096.f);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
constexpr float kLo = 1.f / 4096.f;

// A position in the line of units.
struct Place {
  int r, n, nq, q0;        // sequence, its length, its query tokens and the first one's row
  int unit, units, steps;  // (head, row tile) within the sequence, their count, steps of each
  int step;
};

CKV_DEV int seq_len(const AttArgs& p, int r) {
  const long long cap = (long long)p.a.table_width << p.block_log2;
  return (int)min(min((long long)max(__ldg(p.a.lens + r), 0), cap), (long long)INT32_MAX - 2 * kAttStep);
}
CKV_DEV void seq_queries(const AttArgs& p, int r, int& q0, int& nq) {
  if (p.a.cu) {
    q0 = min(max(__ldg(p.a.cu + r), 0), p.a.tokens);
    nq = min(max(min(__ldg(p.a.cu + r + 1), p.a.tokens) - q0, 0), p.a.max_q);
  } else {
    q0 = r;
    nq = 1;
  }
}
template <int NT> CKV_DEV int seq_units(const AttArgs& p, int nq) {
  return p.c.num_kv_heads * ((nq * p.group + 8 * NT - 1) / (8 * NT));
}
template <int NT> CKV_DEV long long seq_work(const AttArgs& p, int r) {
  int q0, nq;
  seq_queries(p, r, q0, nq);
  return (long long)seq_units<NT>(p, nq) * ((seq_len(p, r) + kAttStep - 1) / kAttStep);
}

// One query row of four floats at p + i in the query's type.
CKV_DEV float4 load_q4(const void* p, int dtype, int64_t i) {
  if (dtype == CKV_FP32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
  float2 x, y;
  if (dtype == CKV_BF16) {
    x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
    y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  } else {
    x = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    y = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  }
  return make_float4(x.x, x.y, y.x, y.y);
}
CKV_DEV void store_out4(void* p, int dtype, int64_t i, float4 v) {
  if (dtype == CKV_FP32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
  } else if (dtype == CKV_BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
}

// Where row `rho` of a unit's sequence and head goes.
CKV_DEV void row_home(const AttArgs& p, int q0, int head, int rho, int64_t& out, int64_t& lse) {
  const int i = rho / p.group, hq = head * p.group + rho % p.group;
  out = (q0 + i) * p.a.out_tok_stride + hq * p.a.out_head_stride;
  lse = (int64_t)(q0 + i) * (p.c.num_kv_heads * p.group) + hq;
}
// The factor on a row's sums and its log-sum-exp, from its maxima (base 2) and its sum.
CKV_DEV float row_factor(float m, float mw, float l) { return l > 0.f || isnan(l) ? exp2f(mw - m) / l : 0.f; }
CKV_DEV float row_lse(float m, float l) { return l > 0.f || isnan(l) ? (m + log2f(l)) * kLn2 : -INFINITY; }

// Merge of `count` partial results of one unit, part(i) their places, by the warps of a CTA
// [w0, w0 + nw): to the output (ctas_left == 0) or to `dst`.
template <int D, int NT, bool kL2, typename F>
CKV_DEV void merge_parts(const AttArgs& p, F part, int count, int w0, int nw, float* dst, int q0, int nq, int head, int tile) {
  constexpr int PER = D / 32;
  auto get = [](const float* x) { return kL2 ? __ldcg(x) : *x; };   // other CTAs' results come from L2
  const int lane = threadIdx.x & 31;
  for (int row = w0; row < 8 * NT; row += nw) {
    const int rho = tile * 8 * NT + row;
    if (!dst && rho >= nq * p.group) break;
    float m = -INFINITY, mw = -INFINITY;
    for (int i = lane; i < count; i += 32) {
      const float* s = part(i) + row * 4;
      m = fmaxf(m, get(s));
      mw = fmaxf(mw, get(s + 1));
    }
    m = warp_max(m);
    mw = warp_max(mw);
    const float m0 = m == -INFINITY ? 0.f : m, mw0 = mw == -INFINITY ? 0.f : mw;
    float l = 0.f, o[PER] = {};
    for (int i = 0; i < count; ++i) {
      const float* s = part(i) + row * 4;
      l += get(s + 2) * exp2f(get(s) - m0);
      const float f = exp2f(get(s + 1) - mw0);
      const float* x = part(i) + 8 * NT * 4 + row * D + lane * PER;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += get(x + e) * f;
    }
    if (dst) {
      if (lane == 0) { dst[row * 4] = m; dst[row * 4 + 1] = mw; dst[row * 4 + 2] = l; }
#pragma unroll
      for (int e = 0; e < PER; ++e) dst[8 * NT * 4 + row * D + lane * PER + e] = o[e];
    } else {
      int64_t at, lat;
      row_home(p, q0, head, rho, at, lat);
      const float f = row_factor(m, mw0, l);
      if constexpr (PER == 4) {
        store_out4(p.a.out, p.a.dtype, at + lane * 4, make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f));
      } else {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __shfl_sync(0xffffffffu, o[e & 1] * f, (2 * lane + (e >> 1)) & 31);
        if (lane < 16) store_out4(p.a.out, p.a.dtype, at + lane * 4, make_float4(v[0], v[1], v[2], v[3]));
      }
      if (p.a.lse && lane == 0) p.a.lse[lat] = row_lse(m, l);
    }
  }
}

struct Entry {     // a piece of a unit that ended in this CTA without being the whole unit
  int used, r, unit, begins, ends;   // begins: the unit's first step is in this piece; ends: its last
  const float* part;
};

template <int D, int kFmt, int NT>
__global__ void __launch_bounds__(kAttWarps * 32, 1) k_attend(const AttArgs p) {
  constexpr int kSteps16 = D / 16;               // k16 steps of the logit product
  constexpr int kDims = D / 8;                   // dims of one lane group, n8 tiles of the output
  constexpr int kStageBytes = 2 * kAttStep * D;  // K then V
  constexpr int kRing = kAttStages * kStageBytes;
  constexpr int kPart = part_floats(D, 8 * NT);
  extern __shared__ __align__(128) char att_smem[];
  __shared__ float s_scale[kAttWarps][kAttStages][4];   // K, V of the step's first and second 16 tokens
  __shared__ Entry s_entry[2 * kAttWarps];
  __shared__ Place s_place[kAttWarps];
  __shared__ int s_scan[32];
  __shared__ long long s_tot[kAttWarps];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, R = p.a.requests;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < 2 * kAttWarps) s_entry[tid].used = 0;
  if (tid < 2) p.desc[cta * 2 + tid] = make_int4(0, 0, 0, 0);

  // ---- the line of units: its length, and where this CTA's warps stand in it
  long long total = 0;
  for (int r = tid; r < R; r += kAttWarps * 32) total += seq_work<NT>(p, r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_tot[wid] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kAttWarps; ++w) total += s_tot[w];
  const int nctas = (int)min((long long)p.ctas, (total + kAttWarps - 1) / kAttWarps);
  const long long c0 = cta < nctas ? total * cta / nctas : total, c1 = cta < nctas ? total * (cta + 1) / nctas : total;
  auto warp_at = [&](int w) { return c0 + (c1 - c0) * w / kAttWarps; };
  long long before = 0;   // work of the sequences before this chunk of threads
  for (int base = 0; base < R; base += kAttWarps * 32) {
    const int r = base + tid;
    const long long mine = r < R ? seq_work<NT>(p, r) : 0;
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_tot[wid] = x;
    __syncthreads();
    long long at = before;
    for (int w = 0; w < wid; ++w) at += s_tot[w];
    for (int w = 0; w < kAttWarps; ++w) before += s_tot[w];
    at += x - mine;
    if (r < R) {
      Place pl;
      pl.r = r;
      pl.n = seq_len(p, r);
      seq_queries(p, r, pl.q0, pl.nq);
      pl.units = seq_units<NT>(p, pl.nq);
      pl.steps = (pl.n + kAttStep - 1) / kAttStep;
      for (int w = 0; w < kAttWarps; ++w) {
        const long long a = warp_at(w);
        if (mine > 0 && a >= at && a < at + mine && a < c1) {
          pl.unit = (int)((a - at) / pl.steps);
          pl.step = (int)((a - at) % pl.steps);
          s_place[w] = pl;
        }
      }
      // sequences with nothing to see: zeros
      if (pl.n == 0 && r % (int)gridDim.x == cta) {
        for (int i = 0; i < pl.nq; ++i)
          for (int hq = 0; hq < p.c.num_kv_heads * p.group; ++hq) {
            const int64_t o = (pl.q0 + i) * p.a.out_tok_stride + hq * p.a.out_head_stride;
            for (int d = 0; d < D; d += 4) store_out4(p.a.out, p.a.dtype, o + d, make_float4(0.f, 0.f, 0.f, 0.f));
            if (p.a.lse) p.a.lse[(int64_t)(pl.q0 + i) * (p.c.num_kv_heads * p.group) + hq] = -INFINITY;
          }
      }
    }
  }
  __syncthreads();

  // ---- this warp's piece
  long long left = warp_at(wid + 1) - warp_at(wid);
  char* ring = att_smem + wid * kRing;
  const uint32_t ring_a = smem_u32(ring), scale_a = smem_u32(&s_scale[wid][0][0]);
  auto swz = [&](int row, int chunk) -> uint32_t {   // 16-byte chunk of a row: no bank conflicts by rows or by columns
    return D == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
  };
  if (left > 0) {
    Place pl = s_place[wid];
    bool first_piece = true;
    while (left > 0) {
      const int todo = (int)min(left, (long long)(pl.steps - pl.step));
      const int s_begin = pl.step, s_end = pl.step + todo;
      const int tiles = pl.units / p.c.num_kv_heads;
      const int head = pl.unit / tiles, tile = pl.unit - head * tiles;
      const int rows = pl.nq * p.group;
      const int n = pl.n;
      const int32_t* table = p.a.tables + pl.r * p.a.table_stride;
      const int pages = (n + (1 << p.block_log2) - 1) >> p.block_log2;
      const char* kh = static_cast<const char*>(p.c.k) + head * p.c.k_head_stride;
      const char* vh = static_cast<const char*>(p.c.v) + head * p.c.v_head_stride;

      // block ids: lane l holds page pbase + l, and the next 32 pages stand by
      int pbase = (s_begin * kAttStep) >> p.block_log2;
      auto page = [&](int i) { return i < pages ? __ldg(table + i) : 0; };
      int pcur = page(pbase + lane), pnext = page(pbase + 32 + lane);
      auto issue = [&](int s, int stage) {
        if (s < s_end) {
          const uint32_t st = ring_a + stage * kStageBytes;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int tok0 = s * kAttStep + half * 16, pi = tok0 >> p.block_log2;
            if (pi - pbase >= 32) {
              pbase += 32;
              pcur = pnext;
              pnext = page(pbase + 32 + lane);
            }
            const int blk = __shfl_sync(0xffffffffu, pcur, pi - pbase);
            const bool good = blk >= 0 && blk < p.c.num_blocks;
            const int64_t b = good ? blk : 0;
            const int off = tok0 & ((1 << p.block_log2) - 1);
            constexpr int kChunks = D / 16, kRows = 32 / kChunks;
            const int row = lane / kChunks, chunk = lane % kChunks;
            const char* ks = kh + b * p.c.k_block_stride + (off + row) * p.c.k_tok_stride + chunk * 16;
            const char* vs = vh + b * p.c.v_block_stride + (off + row) * p.c.v_tok_stride + chunk * 16;
#pragma unroll
            for (int i = 0; i < 16 / kRows; ++i) {
              const bool in = good && tok0 + i * kRows + row < n;
              const uint32_t d = st + swz(half * 16 + i * kRows + row, chunk);
              cp16(d, in ? ks + i * kRows * p.c.k_tok_stride : kh, in ? 16u : 0u);
              cp16(d + kAttStep * D, in ? vs + i * kRows * p.c.v_tok_stride : vh, in ? 16u : 0u);
            }
            if (lane < 2) {
              const float* sc = (lane ? p.c.v_scale : p.c.k_scale) + b * p.c.num_kv_heads + head;
              const uint32_t d = scale_a + (stage * 4 + half * 2 + lane) * 4;
              if (good && tok0 < n) cp4(d, sc);
              else s_scale[wid][stage][half * 2 + lane] = tok0 < n ? __uint_as_float(0x7fffffffu) : 0.f;   // a bad page reads as NaN
            }
          }
        }
        cp_commit();
      };
#pragma unroll
      for (int i = 0; i < kAttStages - 1; ++i) issue(s_begin + i, i);

      // query rows: row g of each tile, split in two fp16 terms
      uint32_t qf[NT][kSteps16][4];
      float qs[NT];           // scale * log2 e * the row's power of two
      int see[NT];            // tokens that the row sees
      int see_min = n;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int rho = (tile * NT + nt) * 8 + g;
        const bool real = rho < rows;
        const int i = rho / p.group, hq = head * p.group + rho % p.group;
        float4 x[kSteps16];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < kSteps16; ++k) {
          const int dim = D == 128 ? (2 * t + k / 4) * 16 + (k & 3) * 4 : t * 16 + k * 4;
          x[k] = real ? load_q4(p.a.q, p.a.dtype, (pl.q0 + i) * p.a.q_tok_stride + hq * p.a.q_head_stride + dim)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
          top = fmaxf(fmaxf(fmaxf(top, fabsf(x[k].x)), fmaxf(fabsf(x[k].y), fabsf(x[k].z))), fabsf(x[k].w));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);   // biased exponent
        const float down = __uint_as_float((uint32_t)(254 - e) << 23);
        qs[nt] = p.a.scale * kLog2e * __uint_as_float((uint32_t)e << 23);
        see[nt] = real && p.a.causal ? n - pl.nq + i + 1 : n;
        see_min = min(see_min, see[nt]);
#pragma unroll
        for (int k = 0; k < kSteps16; ++k) {
          split2(x[k].x * down, x[k].y * down, qf[nt][k][0], qf[nt][k][1]);
          split2(x[k].z * down, x[k].w * down, qf[nt][k][2], qf[nt][k][3]);
        }
      }
      see_min = __reduce_min_sync(0xffffffffu, see_min);

      float o[NT][kDims][2];
      float m[NT], mw[NT], l[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt] = mw[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int j = 0; j < kDims; ++j) o[nt][j][0] = o[nt][j][1] = 0.f;
      }

      int stage = 0;
      for (int s = s_begin; s < s_end; ++s) {
        cp_wait<kAttStages - 2>();
        __syncwarp();
        {
          const int ahead = stage == 0 ? kAttStages - 1 : stage - 1;
          issue(s + kAttStages - 1, ahead);
        }
        const uint32_t kst = ring_a + stage * kStageBytes, vst = kst + kAttStep * D;
        // logits
        float sc[NT][4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[nt][j][0] = sc[nt][j][1] = sc[nt][j][2] = sc[nt][j][3] = 0.f;
          const int row = j * 8 + g;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            const uint4 w = lds4(kst + swz(row, D == 128 ? 2 * t + c : t));
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t b0, b1;
              codes4<kFmt>(ww[e], b0, b1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816(sc[nt][j], qf[nt][c * 4 + e], b0, b1);
            }
          }
        }
        float ks[2], ve[2], vm[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ks[half] = lds1(scale_a + (stage * 4 + half * 2) * 4);
          const float v = lds1(scale_a + (stage * 4 + half * 2 + 1) * 4);
          const uint32_t u = __float_as_uint(v);
          vm[half] = __uint_as_float((u & 0x7fffffu) | 0x3f800000u);
          ve[half] = isnan(v) ? v : (float)((int)(u >> 23 & 255u) - 127);
        }
        const bool masked = (s + 1) * kAttStep > see_min;
        uint32_t pf[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x[4][2], y[4][2];   // logit, and logit + log2 of the value scale (base 2)
          float mn = m[nt], mwn = mw[nt];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float f = qs[nt] * ks[j >> 1];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x[j][e] = fmaf(sc[nt][j][2 + e], kLo, sc[nt][j][e]) * f;
              y[j][e] = x[j][e] + ve[j >> 1];
              if (masked && s * kAttStep + j * 8 + 2 * t + e >= see[nt]) x[j][e] = y[j][e] = -INFINITY;
              mn = fmaxf(mn, x[j][e]);
              mwn = fmaxf(mwn, y[j][e]);
            }
          }
          mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
          mwn = fmaxf(mwn, __shfl_xor_sync(0xffffffffu, mwn, 1));
          mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
          mwn = fmaxf(mwn, __shfl_xor_sync(0xffffffffu, mwn, 2));
          const float m0 = mn == -INFINITY ? 0.f : mn, mw0 = mwn == -INFINITY ? 0.f : mwn;
          if (__any_sync(0xffffffffu, mn > m[nt] || mwn > mw[nt])) {
            l[nt] *= ex2(m[nt] - m0);
            const float f = ex2(mw[nt] - mw0);
#pragma unroll
            for (int j = 0; j < kDims; ++j) { o[nt][j][0] *= f; o[nt][j][1] *= f; }
            m[nt] = mn;
            mw[nt] = mwn;
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
              const int j = 2 * u + jj;
              l[nt] += ex2(x[j][0] - m0) + ex2(x[j][1] - m0);
              const float w0 = ex2(y[j][0] - mw0) * vm[u], w1 = ex2(y[j][1] - mw0) * vm[u];
              split2(w0, w1, pf[nt][u][2 * jj], pf[nt][u][2 * jj + 1]);
            }
        }
        // values: lane (g, t) takes dims g * kDims .. of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each 16
        if constexpr (D == 128) {
          uint4 v[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = lds4(vst + swz(u * 16 + 2 * t + (i & 1) + (i >> 1) * 8, g));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float acc[NT][4][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[nt][k][0] = acc[nt][k][1] = acc[nt][k][2] = acc[nt][k][3] = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t w[4], b0[4], b1[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = e == 0 ? v[u][i].x : e == 1 ? v[u][i].y : e == 2 ? v[u][i].z : v[u][i].w;
              codes4<kFmt>(__byte_perm(w[0], w[1], 0x5140), b0[0], b0[1]);
              codes4<kFmt>(__byte_perm(w[0], w[1], 0x7362), b0[2], b0[3]);
              codes4<kFmt>(__byte_perm(w[2], w[3], 0x5140), b1[0], b1[1]);
              codes4<kFmt>(__byte_perm(w[2], w[3], 0x7362), b1[2], b1[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) mma16816(acc[nt][k], pf[nt][u], b0[k], b1[k]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[nt][e * 4 + k][0] += fmaf(acc[nt][k][2], kLo, acc[nt][k][0]);
                o[nt][e * 4 + k][1] += fmaf(acc[nt][k][3], kLo, acc[nt][k][1]);
              }
          }
        } else {
          uint2 v[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[u][i] = lds2(vst + swz(u * 16 + 2 * t + (i & 1) + (i >> 1) * 8, g >> 1) + (g & 1) * 8);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float acc[NT][4][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[nt][k][0] = acc[nt][k][1] = acc[nt][k][2] = acc[nt][k][3] = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t w[4], b0[4], b1[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = e == 0 ? v[u][i].x : v[u][i].y;
              codes4<kFmt>(__byte_perm(w[0], w[1], 0x5140), b0[0], b0[1]);
              codes4<kFmt>(__byte_perm(w[0], w[1], 0x7362), b0[2], b0[3]);
              codes4<kFmt>(__byte_perm(w[2], w[3], 0x5140), b1[0], b1[1]);
              codes4<kFmt>(__byte_perm(w[2], w[3], 0x7362), b1[2], b1[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) mma16816(acc[nt][k], pf[nt][u], b0[k], b1[k]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[nt][e * 4 + k][0] += fmaf(acc[nt][k][2], kLo, acc[nt][k][0]);
                o[nt][e * 4 + k][1] += fmaf(acc[nt][k][3], kLo, acc[nt][k][1]);
              }
          }
        }
        __syncwarp();   // the stage may be filled again
        stage = stage == kAttStages - 1 ? 0 : stage + 1;
      }
      cp_wait<0>();
      __syncwarp();

      // ---- the piece's end: the whole unit goes out, a part of one is kept for merging
      left -= todo;
      const bool begins = s_begin == 0, ends = s_end == pl.steps;
      float* part = nullptr;
      if (!(begins && ends)) {
        // the ring is free once the warp has no further piece
        part = left > 0 ? p.ws + ((size_t)cta * (kAttWarps + 2) + wid) * kPart : reinterpret_cast<float*>(ring);
        if (lane == 0) {
          Entry& en = s_entry[2 * wid + (first_piece ? 0 : 1)];
          en.used = 1; en.r = pl.r; en.unit = pl.unit; en.begins = begins; en.ends = ends; en.part = part;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float lt = l[nt];
        lt += __shfl_xor_sync(0xffffffffu, lt, 1);
        lt += __shfl_xor_sync(0xffffffffu, lt, 2);
        if (part) {
          const int row = nt * 8 + g;
          if (t == 0) { part[row * 4] = m[nt]; part[row * 4 + 1] = mw[nt]; part[row * 4 + 2] = lt; }
          float4* d = reinterpret_cast<float4*>(part + 8 * NT * 4 + row * D + t * 2 * kDims);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < kDims; j += 4)
              d[(e * kDims + j) / 4] = make_float4(o[nt][j][e], o[nt][j + 1][e], o[nt][j + 2][e], o[nt][j + 3][e]);
        } else {
          const int rho = (tile * NT + nt) * 8 + g;
          if (rho < rows) {
            int64_t at, lat;
            row_home(p, pl.q0, head, rho, at, lat);
            const float f = row_factor(m[nt], mw[nt], lt);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int j = 0; j < kDims; j += 4)
                store_out4(p.a.out, p.a.dtype, at + t * 2 * kDims + e * kDims + j,
                           make_float4(o[nt][j][e] * f, o[nt][j + 1][e] * f, o[nt][j + 2][e] * f, o[nt][j + 3][e] * f));
            if (p.a.lse && t == 0) p.a.lse[lat] = row_lse(m[nt], lt);
          }
        }
      }
      first_piece = false;
      if (left > 0) {   // on to the next unit
        pl.step = 0;
        if (++pl.unit == pl.units) {
          pl.unit = 0;
          do {
            if (++pl.r >= R) { left = 0; break; }   // never expected: keeps the reads in bounds
            pl.n = seq_len(p, pl.r);
            seq_queries(p, pl.r, pl.q0, pl.nq);
            pl.units = seq_units<NT>(p, pl.nq);
            pl.steps = (pl.n + kAttStep - 1) / kAttStep;
          } while (pl.units * pl.steps == 0);
        }
      }
    }
  }
  __syncthreads();

  // ---- merge the pieces of each unit within the CTA
  const float* list[kAttWarps + 1];
  for (int i = 0; i < 2 * kAttWarps;) {
    if (!s_entry[i].used) { ++i; continue; }
    const int r = s_entry[i].r, unit = s_entry[i].unit;
    const bool begins = s_entry[i].begins;
    bool ends = false;
    int count = 0;
    for (; i < 2 * kAttWarps; ++i) {
      if (!s_entry[i].used) continue;
      if (s_entry[i].r != r || s_entry[i].unit != unit) break;
      list[count++] = s_entry[i].part;
      ends = s_entry[i].ends;
    }
    int q0, nq;
    seq_queries(p, r, q0, nq);
    const int tiles = seq_units<NT>(p, nq) / p.c.num_kv_heads;
    const int head = unit / tiles, tile = unit - head * tiles;
    // a unit that reaches past this CTA leaves its part in slot 0 (begun before) or 1
    float* dst = begins && ends ? nullptr : p.ws + ((size_t)cta * (kAttWarps + 2) + kAttWarps + (begins ? 1 : 0)) * kPart;
    merge_parts<D, NT, false>(p, [&](int k) { return list[k]; }, count, wid, kAttWarps, dst, q0, nq, head, tile);
    if (begins && !ends && tid == 0) {
      // the CTA with the unit's last step: the first whose end is at or past the unit's end
      p.desc[cta * 2] = make_int4(1, r, head, tile);
    }
    if (!begins && tid == 0) p.desc[cta * 2 + 1] = make_int4(1, ends ? 1 : 0, 0, 0);
  }
}

// CTA c merges the unit that begins in CTA c of k_attend and reaches past it: its slot 1 and
// slot 0 of the CTAs that follow, up to the one where it ends.
template <int D, int NT>
__global__ void __launch_bounds__(kAttWarps * 32) k_attend_merge(const AttArgs p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kPart = part_floats(D, 8 * NT);
  const int cta = blockIdx.x;
  const int4 d = __ldcg(p.desc + cta * 2);
  if (!d.x) return;
  int count = 1;
  for (int c = cta + 1; c < p.ctas; ++c) {
    const int4 f = __ldcg(p.desc + c * 2 + 1);
    if (!f.x) break;
    ++count;
    if (f.y) break;
  }
  int q0, nq;
  seq_queries(p, d.y, q0, nq);
  merge_parts<D, NT, true>(p, [&](int k) {
    return p.ws + ((size_t)(cta + k) * (kAttWarps + 2) + kAttWarps + (k == 0 ? 1 : 0)) * kPart;
  }, count, threadIdx.x >> 5, kAttWarps, nullptr, q0, nq, d.z, d.w);
}

size_t attention_workspace_bytes(int head_dim, int rows) {
  const int nt = rows > 8 ? 2 : 1;
  return (size_t)kAttMaxCtas * ((kAttWarps + 2) * part_floats(head_dim, 8 * nt) * sizeof(float) + 2 * sizeof(int4));
}

template <int D, int kFmt, int NT>
static cudaError_t att_launch(AttArgs& p, void* ws, cudaStream_t st) {
  constexpr size_t smem = (size_t)kAttWarps * kAttStages * 2 * kAttStep * D;
  static_assert(kAttStages * 2 * kAttStep * D >= part_floats(D, 8 * NT) * 4, "a warp's ring holds one partial result");
  p.ws = static_cast<float*>(ws);
  p.desc = reinterpret_cast<int4*>(p.ws + (size_t)kAttMaxCtas * (kAttWarps + 2) * part_floats(D, 8 * NT));
  auto fn = k_attend<D, kFmt, NT>;
  if (cudaError_t e = ensure_dynamic_smem((const void*)fn, smem); e != cudaSuccess) return e;
  fn<<<p.ctas, kAttWarps * 32, smem, st>>>(p);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(kAttWarps * 32);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_attend_merge<D, NT>, p);
}

template <int D, int kFmt>
static cudaError_t att_pick(AttArgs& p, int rows, void* ws, cudaStream_t st) {
  return rows > 8 ? att_launch<D, kFmt, 2>(p, ws, st) : att_launch<D, kFmt, 1>(p, ws, st);
}

cudaError_t launch_cache_attention(const ckv_cache& c, const ckv_attention_args& a, void* ws, cudaStream_t st) {
  AttArgs p;
  p.c = c;
  p.a = a;
  p.block_log2 = 0;
  while ((1 << p.block_log2) < c.block_size) ++p.block_log2;
  p.group = a.q_heads / c.num_kv_heads;
  p.ctas = kAttMaxCtas;
  const int rows = a.max_q * p.group;
  const bool e4 = c.format == CKV_CACHE_E4M3;
  if (c.head_dim == 64)
    return e4 ? att_pick<64, CKV_CACHE_E4M3>(p, rows, ws, st) : att_pick<64, CKV_CACHE_INT8>(p, rows, ws, st);
  return e4 ? att_pick<128, CKV_CACHE_E4M3>(p, rows, ws, st) : att_pick<128, CKV_CACHE_INT8>(p, rows, ws, st);
}

}  // namespace ckv
