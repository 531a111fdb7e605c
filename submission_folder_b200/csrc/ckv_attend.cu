// Attention of a few query tokens per sequence over the paged 8-bit decode cache.
//
// out = sum_j softmax_j(scale q.k_j) v_j with k_j = ks[b] * ck_j, v_j = vs[b] * cv_j: codes
// c in 8 bits, scales by (block b, KV head).  One pass, with a running maximum.  The scales
// never touch the codes: ks multiplies the logit after its dot product, and vs joins the
// weight as an exponent, w_j = 2^((s_j - m) + log2 vs - m'), which has a reference m' of its own
// on top of the softmax's m; out = 2^m' sum_j w_j c_j / sum_j 2^(s_j - m).  So the matrix products
// run on the codes, which fp16 holds exactly.  s_j - m comes first: m' and log2 vs are small numbers
// and would be lost beside a logit beyond 2^24.
//
// Products: m16n8k16 in fp16 with fp32 sums, tokens (or value dimensions) as the 16 rows of the
// left operand and 8 query rows (a KV head's query heads times the new tokens) as the
// columns, so few rows waste nothing: logits^T = K Q^T, out^T = V^T P^T.  The weights come out
// of the first product with tokens by rows and go into the second with tokens by pairs: one
// 8 x 8 transposition (movmatrix) per 8 tokens.
//
// Precision: a query row is brought to [2^14, 2^15) by a power of two; a bf16 row is exact in fp16,
// fp16 and fp32 rows take two fp16 terms, hi + lo (22 bits).  The weights, at most 2^15, take two terms
// for every type: in one (11 bits) they put a bf16 output off by about 1.4e-4 before its own
// rounding, which flipped the last bit of one output in forty.  The products of one step are summed
// apart and added in fp32 with rounding, because the tensor core's own sums truncate and a warp may
// take thousands of steps.  (Second term and additions for bf16: 1 x 512 tokens 8.7 -> 8.0 us, on fewer warps; 16 ragged
// sequences 20.5 -> 21.7; 32 of up to 32768 tokens 187 -> 192; 131072 tokens x 4 queries 57 -> 71.)
//
// The references m, m' only move when a logit passes them by more than 2^kSlack, so a step
// usually costs one vote instead of the reductions and the rescaling.
//
// Split: the unit of work is 32 tokens of one (sequence, KV head, tile of query rows).  All
// units stand in one line, which is cut evenly into one piece per CTA and then per warp, so a
// ragged batch, a single long sequence and a large batch fill the GPU alike, from lengths
// that only the device knows.  Each warp runs on its own: it copies its tokens' codes with
// cp.async into its own ring of shared memory, a step or two ahead, and multiplies from
// there.  Pieces of one unit are merged in the CTA, then across CTAs by k_attend_merge in
// a fixed order: no atomics, and the same bits every time.
//
// Bound (the kernels alone): HBM (each code is read once for 16 query rows of a KV head) for large
// batches: 32 sequences of up to 32768 tokens, 8 of 32 heads of 128 in bf16: 190 us, 6.0 TB/s.  One
// sequence of 131072 tokens: 51 us with one bf16 query (5.3 TB/s), 71 with four (two row tiles), 123 with
// five (20 rows: two units, each reads and unpacks the codes); 83 us with four fp32 queries, where
// the two terms' products and their sums bound it.  One sequence of 512: 8.1 us, launches and the merges.
#include "ckv_cache.h"
#include "ckv_common.cuh"

namespace ckv {

constexpr int kAttStep = 32;      // tokens per step
constexpr int kAttMaxCtas = 148;
constexpr int kAttMaxWarps = 12;
constexpr float kNone = -3.402823466e38f;   // the reference of a row that has seen nothing: no logit lies below it
constexpr float kSlack = 6.f;     // weights may pass their reference by 2^kSlack
constexpr float kTop = 9.f;       // and stand at 2^kTop there: at most 2^15 in fp16

// Warps and ring stages of a CTA, by what registers and shared memory allow: 8 x 3 steps of
// 8 KB, 8 x 2 where the ring shares shared memory with the query rows of two tiles in two terms.
// 64 dimensions and 8 query rows in one term fit 168 registers: 12 warps (16 sequences of 8192
// tokens: 35 us with 8 warps, 31 with 12; 128 dimensions spill so: 1 x 512 tokens 9.3 us, with 8 warps 7.9).
__host__ __device__ constexpr int att_warps(int D, int nt, int terms) { return D == 64 && nt * terms == 1 ? 12 : 8; }
__host__ __device__ constexpr int att_stages(int nt, int terms) { return nt * terms == 4 ? 2 : 3; }
// Two row tiles in two terms: the query rows (64 registers) stand in shared memory instead, so
// that little spills (131072 tokens x 4 fp32 queries: 91 -> 87 us).
__host__ __device__ constexpr bool att_queries_shared(int nt, int terms) { return nt * terms == 4; }
__host__ __device__ constexpr int att_query_bytes(int nt, int terms, int D) {
  return att_queries_shared(nt, terms) ? nt * terms * (D / 16) * 32 * 8 : 0;   // per warp
}

struct AttArgs {
  ckv_cache c;
  ckv_attention_args a;
  float* ws;                     // [ctas][kAttMaxWarps + 2] partial results
  int4* desc;                    // [ctas]: what k_attend_merge has to merge from this CTA on
  int block_log2, group, ctas;
  int dense;                     // token rows are head_dim bytes apart
  float inv_group;
};

// A partial result: 8 * NT rows of (m, m', l, -) then of D sums.
__host__ __device__ constexpr int part_floats(int D, int rows) { return rows * (D + 4); }

// ---- small pieces -------------------------------------------------------------------
CKV_DEV uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
CKV_DEV void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
CKV_DEV void cp16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {   // bytes 0: zero fill, src not read
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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CKV_DEV void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // d = a b
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 8 x 8 fp16 transposition: lane (g, t) gives (row g, columns 2t, 2t + 1) and gets (rows 2t,
// 2t + 1, column g).
CKV_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
CKV_DEV uint32_t half2_bits(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
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
// (x, y) ~ hi + lo as two fp16 pairs.
CKV_DEV void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = half2_bits(x - f.x, y - f.y);
}

CKV_DEV int seq_len(const AttArgs& p, int r) {
  const long long cap = (long long)p.a.table_width << p.block_log2;
  return (int)min(min((long long)max(p.a.lens[r], 0), cap), (long long)INT32_MAX - 2 * kAttStep);
}
// A sequence's query rows, as many as there are; and those that are computed: none of a sequence that
// has more than max_q.
CKV_DEV void seq_rows(const AttArgs& p, int r, int& q0, int& rows) {
  if (p.a.cu) {
    q0 = min(max(p.a.cu[r], 0), p.a.tokens);
    rows = max(min(p.a.cu[r + 1], p.a.tokens) - q0, 0);
  } else {
    q0 = r;
    rows = 1;
  }
}
CKV_DEV void seq_queries(const AttArgs& p, int r, int& q0, int& nq) {
  seq_rows(p, r, q0, nq);
  if (nq > p.a.max_q) nq = 0;
}
CKV_DEV uint32_t steps_of(int n) { return (uint32_t)(n + kAttStep - 1) / kAttStep; }
template <int NT> CKV_DEV uint32_t seq_units(const AttArgs& p, int nq) {
  return p.c.num_kv_heads * (uint32_t)((nq * p.group + 8 * NT - 1) / (8 * NT));
}
template <int NT> CKV_DEV uint32_t seq_work(const AttArgs& p, int r) {
  int q0, nq;
  seq_queries(p, r, q0, nq);
  return seq_units<NT>(p, nq) * steps_of(seq_len(p, r));
}
// Query token and head within the group of row rho (rho < 2^20: the product cannot reach the
// next whole number).
CKV_DEV void row_split(const AttArgs& p, int rho, int& token, int& member) {
  token = (int)((rho + 0.5f) * p.inv_group);
  member = rho - token * p.group;
}

// x / y for y > 0 by a reciprocal: two rounds leave the quotient within one of the truth.
CKV_DEV uint32_t div_u32(uint32_t x, uint32_t y) {
  const float inv = __frcp_rn((float)y);
  uint32_t q = (uint32_t)(__uint2float_rz(x) * (inv * 0.9999998f));   // below the quotient, by x 2^-21 / y at most
  q += (uint32_t)(__uint2float_rz(x - q * y) * (inv * 0.9999998f));
  return x - q * y >= y ? q + 1 : q;
}

// The line of units cut in `parts`: the first `rem` parts have one step more.
struct Cut {
  uint32_t each, rem;
  CKV_DEV uint32_t at(uint32_t part) const { return part * each + min(part, rem); }
  CKV_DEV uint32_t of(uint32_t x) const {   // the part that holds step x
    const uint32_t big = rem * (each + 1);
    return x < big ? div_u32(x, each + 1) : rem + div_u32(x - big, each);
  }
};

// Four elements, from `dim` on, of a query row in shared memory (chunks of 16 bytes, their
// place turned by the row's low bits g).
CKV_DEV float4 load_q4(uint32_t row, int g, int dtype, int dim) {
  if (dtype == CKV_FP32) {
    const uint4 v = lds4(row + (((dim >> 2) ^ g) << 4));
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
  }
  const uint2 v = lds2(row + (((dim >> 3) ^ g) << 4) + (dim & 4) * 2);
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
  int i, member;
  row_split(p, rho, i, member);
  const int hq = head * p.group + member;
  out = (q0 + i) * p.a.out_tok_stride + hq * p.a.out_head_stride;
  lse = (int64_t)(q0 + i) * (p.c.num_kv_heads * p.group) + hq;
}
// A row's output from its sums, weights' reference (base 2) and weight, and its log-sum-exp.  The
// power of two comes last: it may lie below fp32's range when the values do.
CKV_DEV float4 row_out(float mw, float l, float4 o) {
  const float inv = l > 0.f || isnan(l) ? 1.f / l : 0.f, f = exp2f(mw - kTop);
  return make_float4(o.x * inv * f, o.y * inv * f, o.z * inv * f, o.w * inv * f);
}
CKV_DEV float row_lse(float m, float l) { return l > 0.f || isnan(l) ? (m + log2f(l)) * kLn2 : -INFINITY; }

// A row's running references and sum, and four of its dimensions.
struct RowSum {
  float m = kNone, mw = 0.f, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
};
// Joined by partial results: s their (m, m', l, -), x their sums.
template <int N> CKV_DEV void join(RowSum& a, const float4 (&s)[N], const float4 (&x)[N]) {
  float nm = a.m;
#pragma unroll
  for (int j = 0; j < N; ++j) nm = fmaxf(nm, s[j].x);
  const float kept = a.mw + (a.m - nm);   // references beside the common m
  float nw = kept;
#pragma unroll
  for (int j = 0; j < N; ++j) nw = fmaxf(nw, s[j].y + (s[j].x - nm));
  a.l *= ex2(a.m - nm);
  const float f0 = ex2(kept - nw);
  a.o.x *= f0; a.o.y *= f0; a.o.z *= f0; a.o.w *= f0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    a.l += s[j].z * ex2(s[j].x - nm);
    const float f = ex2(s[j].y + (s[j].x - nm) - nw);
    a.o.x += x[j].x * f; a.o.y += x[j].y * f; a.o.z += x[j].z * f; a.o.w += x[j].w * f;
  }
  a.m = nm;
  a.mw = nw;
}
// Four dimensions, from d on, of row rho of a sequence and head, to the output.
CKV_DEV void store_row(const AttArgs& p, const RowSum& a, int q0, int head, int rho, int d) {
  int64_t at, lat;
  row_home(p, q0, head, rho, at, lat);
  store_out4(p.a.out, p.a.dtype, at + d, row_out(a.mw, a.l, a.o));
  if (p.a.lse && d == 0) p.a.lse[lat] = row_lse(a.m, a.l);
}
constexpr float4 kNoStats = {kNone, 0.f, 0.f, 0.f}, kNoSums = {0.f, 0.f, 0.f, 0.f};

struct Entry {     // a piece of a unit that ended in this CTA without being the whole unit
  int used, q0, rows, head, tile;
  uint32_t begin, end;     // the unit in the line
  const float* part;
};

// NT tiles of 8 query rows share the codes that a warp has converted; kTerms fp16 terms of a query.
template <int D, int kFmt, int NT, int kTerms>
__global__ void __launch_bounds__(att_warps(D, NT, kTerms) * 32, 1) k_attend(const AttArgs p) {
  constexpr int kWarps = att_warps(D, NT, kTerms), kStages = att_stages(NT, kTerms);
  constexpr int kSteps16 = D / 16;               // k16 steps of the logit product
  constexpr int kTiles = D / 16;                 // m16 tiles of the output
  constexpr int kStageBytes = 2 * kAttStep * D;  // K then V
  constexpr int kRing = kStages * kStageBytes;
  constexpr int kAhead = kStages - 1;            // steps in flight during a step's products
  constexpr int kPart = part_floats(D, 8 * NT);
  extern __shared__ __align__(128) char att_smem[];
  __shared__ float s_scale[kWarps][kStages][4];  // K, V of the step's first and second 16 tokens
  __shared__ Entry s_entry[2 * kWarps];
  __shared__ int2 s_group[2 * kWarps];           // of each unit in pieces: its first entry, and all of them as a mask
  __shared__ int s_groups;
  static_assert(2 * kWarps <= 32, "one ballot");
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, R = p.a.requests;
  // each warp clears the entries that it may set itself: no other warp's clearing can come after them
  if (lane < 2) s_entry[2 * wid + lane].used = 0;
  __syncwarp();
  after_previous();

  // ---- the line of units: its length, and where this warp stands in it (each warp for itself)
  const uint32_t first = lane < R ? seq_work<NT>(p, lane) : 0;
  uint32_t total = first;
#pragma unroll 4
  for (int r = lane + 32; r < R; r += 32) total += seq_work<NT>(p, r);
  total = __reduce_add_sync(0xffffffffu, total);
  const uint32_t nctas = min((uint32_t)p.ctas, (total + kWarps - 1) / kWarps);
  const uint32_t per_cta = nctas ? div_u32(total, nctas) : 0u;
  const Cut cut = {per_cta, total - per_cta * nctas};
  const uint32_t c0 = cta < nctas ? cut.at(cta) : total, c1 = cta < nctas ? cut.at(cta + 1) : total;
  const Cut warps = {(c1 - c0) / kWarps, (c1 - c0) % kWarps};
  const uint32_t here = c0 + warps.at(wid);
  uint32_t left = warps.at(wid + 1) - warps.at(wid);
  int r = 0;
  uint32_t seq_at = 0;   // where sequence r begins in the line
  if (left > 0) {
    for (int base = 0; base < R; base += 32) {
      const uint32_t mine = base == 0 ? first : base + lane < R ? seq_work<NT>(p, base + lane) : 0;
      const uint32_t sum = __reduce_add_sync(0xffffffffu, mine);
      if (here >= seq_at + sum) { seq_at += sum; continue; }
      uint32_t x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const int at = __ffs(__ballot_sync(0xffffffffu, here < seq_at + x)) - 1;
      r = base + at;
      seq_at += __shfl_sync(0xffffffffu, x - mine, at);
      break;
    }
  }

  // ---- this warp's piece
  char* ring = att_smem + wid * kRing;
  const uint32_t ring_a = smem_u32(ring), scale_a = smem_u32(&s_scale[wid][0][0]);
  // 16-byte chunk of a row, so that neither reads by rows nor reads by columns meet in a bank
  auto swz = [&](int row, int chunk) -> uint32_t {
    return D == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
  };
  constexpr int kChunks = D / 16, kRows = 32 / kChunks;   // of one copy instruction
  // from the place of row crow to that of row crow + i * kRows (kRows = 4 at D = 128: every second turns
  // the chunk's third bit; 8 at D = 64: the swizzle is the same)
  auto turn = [&](int i) -> uint32_t {
    const uint32_t here = swz(lane / kChunks, lane % kChunks), there = swz(lane / kChunks + i * kRows, lane % kChunks);
    return there - here;
  };
  const int crow = lane / kChunks, cchunk = lane % kChunks;
  if (left > 0) {
    int n = seq_len(p, r), q0, nq;
    seq_queries(p, r, q0, nq);
    uint32_t steps = steps_of(n);
    uint32_t unit = div_u32(here - seq_at, steps);
    int step = (int)(here - seq_at - unit * steps);
    bool first_piece = true;
    while (left > 0) {
      const int todo = (int)min(left, steps - step);
      const int s_begin = step, s_end = step + todo;
      const uint32_t tiles = (uint32_t)(nq * p.group + 8 * NT - 1) / (8 * NT);
      const int head = tiles == 1 ? unit : div_u32(unit, tiles), tile = unit - head * tiles;
      const int rows = nq * p.group;
      const int32_t* table = p.a.tables + r * p.a.table_stride;
      const int pages = (n + (1 << p.block_log2) - 1) >> p.block_log2;
      const char* kh = static_cast<const char*>(p.c.k) + head * p.c.k_head_stride + crow * p.c.k_tok_stride + cchunk * 16;
      const char* vh = static_cast<const char*>(p.c.v) + head * p.c.v_head_stride + crow * p.c.v_tok_stride + cchunk * 16;

      // block ids: lane l holds page pbase + l, and the next 32 pages stand by
      int pbase = (s_begin * kAttStep) >> p.block_log2;
      auto page = [&](int i) { return i < pages ? table[i] : 0; };
      int pcur = page(pbase + lane), pnext = page(pbase + 32 + lane);
      // the 32 tokens of step s, as two halves of 16 that may stand in two blocks
      auto issue = [&](int s, int stage) {
        const int tok0 = s * kAttStep, tok1 = tok0 + 16, last = (1 << p.block_log2) - 1;
        if ((tok0 >> p.block_log2) - pbase >= 32) {   // pbase is even where a step has two pages
          pbase += 32;
          pcur = pnext;
          pnext = page(pbase + 32 + lane);
        }
        const int blk0 = __shfl_sync(0xffffffffu, pcur, (tok0 >> p.block_log2) - pbase);
        const int blk1 = __shfl_sync(0xffffffffu, pcur, (tok1 >> p.block_log2) - pbase);
        const bool good0 = (uint32_t)blk0 < (uint32_t)p.c.num_blocks, good1 = (uint32_t)blk1 < (uint32_t)p.c.num_blocks;
        const uint32_t st = ring_a + stage * kStageBytes + swz(crow, cchunk);
        if (p.dense && good0 && good1 && tok0 + kAttStep <= n) {   // rows D bytes apart: constant offsets
          const char* k0 = kh + (uint64_t)(uint32_t)blk0 * p.c.k_block_stride + (tok0 & last) * D;
          const char* v0 = vh + (uint64_t)(uint32_t)blk0 * p.c.v_block_stride + (tok0 & last) * D;
          const char* k1 = k0 + 16 * D;
          const char* v1 = v0 + 16 * D;
          if (p.block_log2 == 4) {
            k1 = kh + (uint64_t)(uint32_t)blk1 * p.c.k_block_stride;
            v1 = vh + (uint64_t)(uint32_t)blk1 * p.c.v_block_stride;
          }
#pragma unroll
          for (int i = 0; i < 16 / kRows; ++i) {   // the swizzle repeats every 8 rows
            const uint32_t d = st + turn(i);
            cp16(d, k0 + i * kRows * D);
            cp16(d + 16 * D, k1 + i * kRows * D);
            cp16(d + kAttStep * D, v0 + i * kRows * D);
            cp16(d + kAttStep * D + 16 * D, v1 + i * kRows * D);
          }
        } else {
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            const int tok = half ? tok1 : tok0;
            const bool good = half ? good1 : good0;
            const int64_t b = good ? (half ? blk1 : blk0) : 0;
            const int have = good ? n - tok : 0;   // rows of these 16 that hold tokens
            const char* ks = kh + b * p.c.k_block_stride + (tok & last) * p.c.k_tok_stride;
            const char* vs = vh + b * p.c.v_block_stride + (tok & last) * p.c.v_tok_stride;
#pragma unroll
            for (int i = 0; i < 16 / kRows; ++i) {
              const uint32_t in = i * kRows + crow < have ? 16u : 0u;
              const uint32_t d = st + turn(i) + half * 16 * D;
              cp16_or_zero(d, in ? ks + i * kRows * p.c.k_tok_stride : kh, in);
              cp16_or_zero(d + kAttStep * D, in ? vs + i * kRows * p.c.v_tok_stride : vh, in);
            }
          }
        }
        if (lane < 4) {   // scales: K, V of each half; a bad page reads as NaN
          const int blk = lane < 2 ? blk0 : blk1;
          const float* from = (lane & 1 ? p.c.v_scale : p.c.k_scale) + (int64_t)blk * p.c.num_kv_heads + head;
          if ((lane < 2 ? tok0 : tok1) >= n) s_scale[wid][stage][lane] = 0.f;
          else if (lane < 2 ? good0 : good1) cp4(scale_a + (stage * 4 + lane) * 4, from);
          else s_scale[wid][stage][lane] = __uint_as_float(0x7fffffffu);
        }
      };

      constexpr bool kShared = att_queries_shared(NT, kTerms);
      uint32_t qf[kShared ? 1 : NT][kShared ? 1 : kTerms][kShared ? 1 : kSteps16][2];
      const uint32_t qf_a = smem_u32(att_smem) + kWarps * kRing + wid * att_query_bytes(NT, kTerms, D) + lane * 16;
      float qs[NT][2];        // rows 2t, 2t + 1: scale * log2 e * the row's power of two
      int see[NT][2];         // tokens that they see
      int see_min = n;
      // the query rows come through the ring's last stage, ahead of the first codes
      const uint32_t q_a = ring_a + kAhead * kStageBytes;
      const int q_log2 = (D == 128 ? 4 : 3) + (p.a.dtype == CKV_FP32 ? 1 : 0);   // 16-byte chunks of a row
      auto copy_chunk = [&](int i) {
        const int row = i >> q_log2, chunk = i & ((1 << q_log2) - 1), rho = tile * NT * 8 + row;
        int tok, member;
        row_split(p, rho, tok, member);
        const char* src = static_cast<const char*>(p.a.q) +
                          ((q0 + tok) * p.a.q_tok_stride + (head * p.group + member) * p.a.q_head_stride) * (p.a.dtype == CKV_FP32 ? 4 : 2);
        cp16_or_zero(q_a + (row << q_log2 << 4) + ((chunk ^ (row & 7)) << 4), rho < rows ? src + chunk * 16 : p.a.q, rho < rows ? 16u : 0u);
      };
      if constexpr (kShared) {   // side by side where the registers allow it (131072 x 4 queries: 87 -> 85 us)
#pragma unroll 4
        for (int i = lane; i < 8 * NT << q_log2; i += 32) copy_chunk(i);
      } else {
        for (int i = lane; i < 8 * NT << q_log2; i += 32) copy_chunk(i);
      }
      cp_commit();
      // lane (g, t) has row g's dimensions of its chunks
      auto load_queries = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int rho = (tile * NT + nt) * 8 + g;
          const uint32_t row = q_a + ((nt * 8 + g) << q_log2 << 4);
          auto dim_of = [&](int k) { return D == 128 ? (2 * t + k / 4) * 16 + (k & 3) * 4 : t * 16 + k * 4; };
          float top;
          float4 x[kSteps16];
          uint2 w[kSteps16];
          if constexpr (kTerms == 1) {   // bf16: magnitudes of both halves of a word at a time
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < kSteps16; ++k) {
              w[k] = lds2(row + (((dim_of(k) >> 3) ^ g) << 4) + (dim_of(k) & 4) * 2);
              asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[k].x));
              asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[k].y));
            }
            top = fmaxf(fabsf(__uint_as_float(m << 16)), fabsf(__uint_as_float(m & 0xffff0000u)));
          } else {
            top = 0.f;
#pragma unroll
            for (int k = 0; k < kSteps16; ++k) {
              x[k] = load_q4(row, g, p.a.dtype, dim_of(k));
              top = fmaxf(fmaxf(fmaxf(top, fabsf(x[k].x)), fmaxf(fabsf(x[k].y), fabsf(x[k].z))), fabsf(x[k].w));
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // the row times 2^(14 - exponent); exponents at the ends of the range are clamped
          const int e = min(max((int)(__float_as_uint(top) >> 23), 16), 254);   // biased
          const float up = __uint_as_float((uint32_t)(268 - e) << 23);
          const float mine = p.a.scale * kLog2e * __uint_as_float((uint32_t)(e - 14) << 23);   // over up
          int i, member;
          row_split(p, rho, i, member);
          const int sees = rho < rows && p.a.causal ? n - nq + i + 1 : n;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            qs[nt][r] = __shfl_sync(0xffffffffu, mine, (2 * t + r) * 4);
            see[nt][r] = __shfl_sync(0xffffffffu, sees, (2 * t + r) * 4);
            see_min = min(see_min, see[nt][r]);
          }
#pragma unroll
          for (int k = 0; k < kSteps16; ++k) {
            if constexpr (kTerms == 1) {
              auto to_half = [&](uint32_t v) {
                return half2_bits(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xffff0000u) * up);
              };
              qf[nt][0][k][0] = to_half(w[k].x);
              qf[nt][0][k][1] = to_half(w[k].y);
            } else {
              uint32_t f[2][2];   // [term][pair]
              split2(x[k].x * up, x[k].y * up, f[0][0], f[1][0]);
              split2(x[k].z * up, x[k].w * up, f[0][1], f[1][1]);
              if constexpr (kShared) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(qf_a + (k * NT + nt) * 512), "r"(f[0][0]),
                             "r"(f[0][1]), "r"(f[1][0]), "r"(f[1][1]) : "memory");
              } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  qf[nt][0][k][i] = f[0][i];
                  qf[nt][1][k][i] = f[1][i];
                }
              }
            }
          }
        }
        see_min = __reduce_min_sync(0xffffffffu, see_min);
      };

      // out^T: tile i has dims (g * kTiles * 2 + 2 i, + 1) x rows (2t, 2t + 1)
      float o[NT][kTiles][4];
      float m[NT][2], mw[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 2; ++r) { m[nt][r] = l[nt][r] = 0.f; mw[nt][r] = kNone; }   // kNone: m is not set yet
#pragma unroll
        for (int j = 0; j < kTiles; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      }

      int fill = 0, stage = 0;   // ring stages to fill and to use next
#pragma unroll 1
      for (int s = s_begin - kAhead; s < s_end; ++s) {   // one copy of the code for the ring's filling and its use
        if (s + kAhead < s_end) issue(s + kAhead, fill);
        cp_commit();
        fill = fill == kStages - 1 ? 0 : fill + 1;
        if (s + kAhead == s_begin) {
          cp_wait<1>();
          __syncwarp();
          load_queries();
          __syncwarp();
        }
        if (s < s_begin) continue;
        cp_wait<kAhead>();
        __syncwarp();
        const uint32_t kst = ring_a + stage * kStageBytes, vst = kst + kAttStep * D;
        // logits^T: lane holds tokens g, g + 8 of each 16 x rows 2t, 2t + 1
        float sc[NT][2][4];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint4 w[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[u][h] = lds4(kst + swz(u * 16 + h * 8 + g, D == 128 ? 2 * t + c : t));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              codes4<kFmt>(e == 0 ? w[u][0].x : e == 1 ? w[u][0].y : e == 2 ? w[u][0].z : w[u][0].w, a[u][0], a[u][2]);
              codes4<kFmt>(e == 0 ? w[u][1].x : e == 1 ? w[u][1].y : e == 2 ? w[u][1].z : w[u][1].w, a[u][1], a[u][3]);
            }
            uint32_t b[NT][kTerms][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if constexpr (kShared) {
                const uint4 v = lds4(qf_a + ((c * 4 + e) * NT + nt) * 512);
                b[nt][0][0] = v.x; b[nt][0][1] = v.y; b[nt][1][0] = v.z; b[nt][1][1] = v.w;
              } else {
#pragma unroll
                for (int k = 0; k < kTerms; ++k) { b[nt][k][0] = qf[nt][k][c * 4 + e][0]; b[nt][k][1] = qf[nt][k][c * 4 + e][1]; }
              }
            }
            // the sums of the 16-token halves and the row tiles are independent: they take turns
#pragma unroll
            for (int k = 0; k < kTerms; ++k)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  if (c == 0 && e == 0 && k == 0) mma16816_zero(sc[nt][u], a[u], b[nt][k][0], b[nt][k][1]);
                  else mma16816(sc[nt][u], a[u], b[nt][k][0], b[nt][k][1]);
                }
          }
        }
        float ks[2], ve[2], top[2];   // top: kTop, or NaN where the value scale is one
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ks[u] = lds1(scale_a + (stage * 4 + u * 2) * 4);
          const float v = lds1(scale_a + (stage * 4 + u * 2 + 1) * 4);
          const uint32_t bits = __float_as_uint(v), mant = bits & 0x7fffffu;
          ve[u] = (float)((int)(bits >> 23 & 255u) - 127);
          if (mant) ve[u] += __log2f(__uint_as_float(mant | 0x3f800000u));   // not a power of two
          top[u] = isnan(v) ? v : kTop;
        }
        float over[NT][2][2];   // log2 vs over the weights' reference, ready before the vote (x 4 fp32 queries 83.5 -> 82.6 us)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u) over[nt][r][u] = ve[u] - mw[nt][r];
        bool hide = false;   // a token that a row does not see stands in a block whose value scale is NaN
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float f = qs[nt][r] * ks[u];   // logits relative to m, rounded once
              sc[nt][u][r] = fmaf(sc[nt][u][r], f, -m[nt][r]);
              sc[nt][u][2 + r] = fmaf(sc[nt][u][2 + r], f, -m[nt][r]);
            }
        if ((s + 1) * kAttStep > see_min) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (s * kAttStep + u * 16 + g + (e >> 1) * 8 >= see[nt][e & 1]) sc[nt][u][e] = -INFINITY;
          hide = isnan(top[0]) || isnan(top[1]);
        }
        bool past = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float h0 = fmaxf(sc[nt][0][r], sc[nt][0][2 + r]), h1 = fmaxf(sc[nt][1][r], sc[nt][1][2 + r]);
            past = past || fmaxf(h0, h1) > kSlack || fmaxf(h0 + over[nt][r][0], h1 + over[nt][r][1]) > kSlack;
          }
        if (__any_sync(0xffffffffu, past)) {
          float shift[NT][2];
          // the rows that passed theirs get new references (whole numbers: the rescaling is exact),
          // the same in all lanes of a row and whatever the other rows do
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float h0 = fmaxf(sc[nt][0][r], sc[nt][0][2 + r]), h1 = fmaxf(sc[nt][1][r], sc[nt][1][2 + r]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) {
                h0 = fmaxf(h0, __shfl_xor_sync(0xffffffffu, h0, d));
                h1 = fmaxf(h1, __shfl_xor_sync(0xffffffffu, h1, d));
              }
              // the first logit that a row sees sets m; rounded up, so that none stays above it
              const bool unset = mw[nt][r] == kNone, move = unset ? fmaxf(h0, h1) > -INFINITY : fmaxf(h0, h1) > kSlack;
              const float nm = move ? ceilf(__fadd_ru(m[nt][r], fmaxf(h0, h1))) : m[nt][r], d = nm - m[nt][r];
              const float kept = mw[nt][r] - d;   // the old reference of the weights beside the new m
              float nw = fmaxf(h0 - d + ve[0], h1 - d + ve[1]);
              nw = nw > kept + kSlack ? ceilf(nw) : kept;
              l[nt][r] *= unset ? 1.f : ex2(-d);   // not set: nothing but zeros or a NaN
              const float f = ex2(kept - nw);
              m[nt][r] = nm;
              mw[nt][r] = nw;
              over[nt][r][0] = ve[0] - nw;
              over[nt][r][1] = ve[1] - nw;
#pragma unroll
              for (int j = 0; j < kTiles; ++j) { o[nt][j][r] *= f; o[nt][j][2 + r] *= f; }
              shift[nt][r] = d;
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int u = 0; u < 2; ++u) { sc[nt][u][r] -= shift[nt][r]; sc[nt][u][2 + r] -= shift[nt][r]; }
        }
        uint32_t pf[NT][2][2][2];   // [term]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = e & 1;
              l[nt][r] += ex2(sc[nt][u][e]);
              w[e] = ex2(sc[nt][u][e] + (over[nt][r][u] + top[u]));
            }
            if (hide) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (sc[nt][u][e] == -INFINITY) w[e] = 0.f;
            }
            uint32_t h0, l0, h1, l1;
            split2(w[0], w[1], h0, l0);
            split2(w[2], w[3], h1, l1);
            pf[nt][0][u][0] = transpose8(h0);
            pf[nt][0][u][1] = transpose8(h1);
            pf[nt][1][u][0] = transpose8(l0);
            pf[nt][1][u][1] = transpose8(l1);
          }
        // values: lane (g, t) takes dims g * 2 kTiles .. of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each 16
        uint32_t v[2][4][D / 32];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = u * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
            if constexpr (D == 128) {
              const uint4 q = lds4(vst + swz(row, g));
              v[u][i][0] = q.x; v[u][i][1] = q.y; v[u][i][2] = q.z; v[u][i][3] = q.w;
            } else {
              const uint2 q = lds2(vst + swz(row, g >> 1) + (g & 1) * 8);
              v[u][i][0] = q.x; v[u][i][1] = q.y;
            }
          }
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {   // 4 dims, two tiles
          uint32_t a[2][2][4];               // [u][tile]
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h ? 0x7362 : 0x5140;
              codes4<kFmt>(__byte_perm(v[u][0][e], v[u][1][e], sel), a[u][h][0], a[u][h][1]);
              codes4<kFmt>(__byte_perm(v[u][2][e], v[u][3][e], sel), a[u][h][2], a[u][h][3]);
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float(&acc)[4] = o[nt][2 * e + h];
              float d[4];
              mma16816_zero(d, a[0][h], pf[nt][1][0][0], pf[nt][1][0][1]);
              mma16816(d, a[1][h], pf[nt][1][1][0], pf[nt][1][1][1]);
              mma16816(d, a[0][h], pf[nt][0][0][0], pf[nt][0][0][1]);
              mma16816(d, a[1][h], pf[nt][0][1][0], pf[nt][0][1][1]);
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[k] += d[k];
            }
        }
        __syncwarp();   // the stage may be filled again
        stage = stage == kStages - 1 ? 0 : stage + 1;
      }
      cp_wait<0>();
      __syncwarp();

      // ---- the piece's end: the whole unit goes out, a part of one is kept for merging
      left -= todo;
      float* part = nullptr;
      if (todo != (int)steps) {
        // the ring is free once the warp has no further piece
        part = left > 0 ? p.ws + ((size_t)cta * (kAttMaxWarps + 2) + wid) * kPart : reinterpret_cast<float*>(ring);
        if (lane == 0) {
          Entry& en = s_entry[2 * wid + (first_piece ? 0 : 1)];
          en.used = 1; en.q0 = q0; en.rows = rows; en.head = head; en.tile = tile; en.part = part;
          en.begin = seq_at + unit * steps;
          en.end = en.begin + steps;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float lt = l[nt][r];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, d);
          const int row = nt * 8 + 2 * t + r;
          if (part) {
            const bool unset = mw[nt][r] == kNone;
            if (g == 0) *reinterpret_cast<float4*>(part + row * 4) = make_float4(unset ? kNone : m[nt][r], unset ? 0.f : mw[nt][r], lt, 0.f);
            float4* d = reinterpret_cast<float4*>(part + 8 * NT * 4 + row * D + g * 2 * kTiles);
#pragma unroll
            for (int j = 0; j < kTiles; j += 2)
              d[j / 2] = make_float4(o[nt][j][r], o[nt][j][2 + r], o[nt][j + 1][r], o[nt][j + 1][2 + r]);
          } else {
            const int rho = tile * NT * 8 + row;
            if (rho < rows) {
              int64_t at, lat;
              row_home(p, q0, head, rho, at, lat);
#pragma unroll
              for (int j = 0; j < kTiles; j += 2)
                store_out4(p.a.out, p.a.dtype, at + g * 2 * kTiles + 2 * j,
                           row_out(mw[nt][r], lt, make_float4(o[nt][j][r], o[nt][j][2 + r], o[nt][j + 1][r], o[nt][j + 1][2 + r])));
              if (p.a.lse && g == 0) p.a.lse[lat] = row_lse(m[nt][r], lt);
            }
          }
        }
      first_piece = false;
      if (left > 0) {   // on to the next unit
        step = 0;
        if (++unit == p.c.num_kv_heads * tiles) {
          seq_at += unit * steps;
          unit = 0;
          do {
            if (++r >= R) { left = 0; break; }   // never expected: keeps the reads in bounds
            n = seq_len(p, r);
            seq_queries(p, r, q0, nq);
            steps = steps_of(n);
          } while (nq * steps == 0);
        }
      }
    }
  }
  __syncthreads();

  // ---- merge the pieces of each unit within the CTA; a unit that reaches past the CTA leaves its
  // part in slot 0 (begun in a CTA before) or 1 (begun here)
  if (c1 > c0) {
    if (wid == 0) {
      const bool used = lane < 2 * kWarps && s_entry[lane].used;
      const uint32_t mask = __ballot_sync(0xffffffffu, used), below = mask & ((1u << lane) - 1);
      const uint32_t mine = used ? s_entry[lane].begin : 0;
      const uint32_t prev = __shfl_sync(0xffffffffu, mine, below ? 31 - __clz(below) : 0);
      const bool first_of = used && (!below || prev != mine);
      const uint32_t firsts = __ballot_sync(0xffffffffu, first_of);
      const uint32_t later = lane < 31 ? firsts >> (lane + 1) << (lane + 1) : 0;
      if (first_of)
        s_group[__popc(firsts & ((1u << lane) - 1))] =
            make_int2(lane, mask & (0xffffffffu << lane) & (later ? (later & -later) - 1 : 0xffffffffu));
      if (lane == 0) s_groups = __popc(firsts);
    }
    __syncthreads();
    const int groups = s_groups;
    // a warp has a row of a unit: lane i the references and sum of piece i, then four dimensions
    for (int i = wid; i < groups * 8 * NT; i += kWarps) {
      const int row = i / groups, grp = i - row * groups, d = lane * 4;
      const Entry& e = s_entry[s_group[grp].x];
      if (e.tile * 8 * NT + row >= e.rows) continue;
      uint32_t list = s_group[grp].y;
      const bool begins = e.begin >= c0, ends = e.end <= c1, mine = list >> lane & 1u;
      const unsigned long long my_part = mine ? reinterpret_cast<unsigned long long>(s_entry[lane].part) : 0;
      const float4 st = mine ? *(reinterpret_cast<const float4*>(my_part) + row) : kNoStats;
      RowSum sum;
      sum.m = st.x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) sum.m = fmaxf(sum.m, __shfl_xor_sync(0xffffffffu, sum.m, o));
      const float kept = st.y + (st.x - sum.m);
      sum.mw = kept;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) sum.mw = fmaxf(sum.mw, __shfl_xor_sync(0xffffffffu, sum.mw, o));
      sum.l = st.z * ex2(st.x - sum.m);
      const float f = ex2(kept - sum.mw);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) sum.l += __shfl_xor_sync(0xffffffffu, sum.l, o);
      while (list) {   // four pieces at a time, ascending
        float4 x[4];
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int piece = list ? __ffs(list) - 1 : 0;
          const float* part = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, my_part, piece));
          w[j] = __shfl_sync(0xffffffffu, f, piece);
          x[j] = kNoSums;
          if (list && d < D) x[j] = *reinterpret_cast<const float4*>(part + 8 * NT * 4 + row * D + d);
          list &= list - 1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum.o.x += x[j].x * w[j]; sum.o.y += x[j].y * w[j]; sum.o.z += x[j].z * w[j]; sum.o.w += x[j].w * w[j];
        }
      }
      if (d >= D) continue;
      if (begins && ends) {
        store_row(p, sum, e.q0, e.head, e.tile * 8 * NT + row, d);
      } else {
        float* dst = p.ws + ((size_t)cta * (kAttMaxWarps + 2) + kAttMaxWarps + (begins ? 1 : 0)) * kPart;
        if (d == 0) *reinterpret_cast<float4*>(dst + row * 4) = make_float4(sum.m, sum.mw, sum.l, 0.f);
        *reinterpret_cast<float4*>(dst + 8 * NT * 4 + row * D + d) = sum.o;
      }
    }
    if (tid == kWarps * 32 - 1) {   // the last unit may reach past the CTA
      int4 todo = make_int4(0, 0, 0, 0);
      if (groups) {
        const Entry& e = s_entry[s_group[groups - 1].x];
        if (e.begin >= c0 && e.end > c1) todo = make_int4((int)(cut.of(e.end - 1) - cta + 1) | e.head << 8, e.q0, e.rows, e.tile);
      }
      p.desc[cta] = todo;
    }
  } else if (tid == 0) {
    p.desc[cta] = make_int4(0, 0, 0, 0);
  }

  // log-sum-exp of rows of no sequence
  if (p.a.lse && p.a.cu) {
    const int64_t hq = p.c.num_kv_heads * p.group;
    for (int64_t i = max(p.a.cu[R], 0) * hq + cta * kWarps * 32 + tid; i < p.a.tokens * hq; i += (int64_t)gridDim.x * kWarps * 32)
      p.a.lse[i] = -INFINITY;
  }
  // sequences with nothing to see: zeros; with more rows than max_q: NaN
  for (int r = cta; r < R; r += gridDim.x) {
    int q0, rows;
    seq_rows(p, r, q0, rows);
    const bool empty = seq_len(p, r) == 0, many = !empty && rows > p.a.max_q;
    if (!empty && !many) continue;
    const int hq = p.c.num_kv_heads * p.group;
    const float x = many ? __uint_as_float(0x7fffffffu) : 0.f;
    for (int tok = q0; tok < q0 + rows; ++tok)
      for (int i = tid; i < hq * (D / 4); i += kWarps * 32) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        store_out4(p.a.out, p.a.dtype, tok * p.a.out_tok_stride + h * p.a.out_head_stride + d, make_float4(x, x, x, x));
        if (p.a.lse && d == 0) p.a.lse[(int64_t)tok * hq + h] = many ? x : -INFINITY;
      }
  }
}

// CTA c merges the unit that begins in CTA c of k_attend and reaches past it: its slot 1 and
// slot 0 of the CTAs that follow, up to the one where it ends.  A thread has four dimensions of
// a row; the parts go round kGroups groups of threads, whose sums meet in shared memory (one
// group: 131072 tokens x 4 fp32 queries 84 us in all, 80 so).
constexpr int kMergeThreads = 1024;

template <int D, int NT>
__global__ void __launch_bounds__(kMergeThreads) k_attend_merge(const AttArgs p) {
  constexpr int kPart = part_floats(D, 8 * NT), kItems = 8 * NT * (D / 4), kGroups = kMergeThreads / kItems, kBatch = 4;
  __shared__ float4 s_stats[kMergeThreads], s_sums[kMergeThreads];
  after_previous();
  const int cta = blockIdx.x, item = threadIdx.x % kItems, grp = threadIdx.x / kItems;
  const int row = item / (D / 4), d = item % (D / 4) * 4;
  auto load = [&](int k, float4& s, float4& x) {
    const float* part = p.ws + ((size_t)(cta + k) * (kAttMaxWarps + 2) + kAttMaxWarps + (k == 0 ? 1 : 0)) * kPart;
    s = *reinterpret_cast<const float4*>(part + row * 4);
    x = *reinterpret_cast<const float4*>(part + 8 * NT * 4 + row * D + d);
  };
  // a group's first part is read before it is known whether there is one
  float4 s0[1] = {kNoStats}, x0[1] = {kNoSums};
  if (cta + grp < p.ctas) load(grp, s0[0], x0[0]);
  const int4 unit = p.desc[cta];   // parts | head << 8, first query token, rows, tile
  if (!unit.x) return;
  const int parts = unit.x & 255, rho = unit.w * 8 * NT + row;
  RowSum sum;
  if (grp < parts) join(sum, s0, x0);
  for (int k = grp + kGroups; k < parts; k += kGroups * kBatch) {
    float4 s[kBatch], x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      s[j] = kNoStats;
      x[j] = kNoSums;
      if (k + j * kGroups < parts) load(k + j * kGroups, s[j], x[j]);
    }
    join(sum, s, x);
  }
  if constexpr (kGroups > 1) {
    if (grp > 0) {
      s_stats[threadIdx.x] = make_float4(sum.m, sum.mw, sum.l, 0.f);
      s_sums[threadIdx.x] = sum.o;
    }
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      s0[0] = s_stats[g * kItems + item];
      x0[0] = s_sums[g * kItems + item];
      join(sum, s0, x0);
    }
  }
  if (rho < unit.z) store_row(p, sum, unit.y, unit.x >> 8, rho, d);
}

size_t attention_workspace_bytes(int head_dim, int rows) {
  const int nt = rows > 8 ? 2 : 1;
  return (size_t)kAttMaxCtas * ((kAttMaxWarps + 2) * part_floats(head_dim, 8 * nt) * sizeof(float) + sizeof(int4));
}

template <int D, int kFmt, int NT, int kTerms>
static cudaError_t att_launch(AttArgs& p, void* ws, cudaStream_t st) {
  constexpr size_t smem = (size_t)att_warps(D, NT, kTerms) * (att_stages(NT, kTerms) * 2 * kAttStep * D + att_query_bytes(NT, kTerms, D));
  static_assert(att_stages(NT, kTerms) * 2 * kAttStep * D >= part_floats(D, 8 * NT) * 4, "a warp's ring holds one partial result");
  static_assert(att_warps(D, NT, kTerms) <= kAttMaxWarps, "workspace slots");
  p.ws = static_cast<float*>(ws);
  p.desc = reinterpret_cast<int4*>(p.ws + (size_t)kAttMaxCtas * (kAttMaxWarps + 2) * part_floats(D, 8 * NT));
  auto fn = k_attend<D, kFmt, NT, kTerms>;
  if (cudaError_t e = ensure_dynamic_smem((const void*)fn, smem); e != cudaSuccess) return e;
  if (cudaError_t e = launch_after(fn, dim3(p.ctas), att_warps(D, NT, kTerms) * 32, smem, st, p); e != cudaSuccess) return e;
  return launch_after(k_attend_merge<D, NT>, dim3(p.ctas), kMergeThreads, 0, st, p);
}

template <int D, int kFmt>
static cudaError_t att_pick(AttArgs& p, int rows, void* ws, cudaStream_t st) {
  if (p.a.dtype == CKV_BF16) return rows > 8 ? att_launch<D, kFmt, 2, 1>(p, ws, st) : att_launch<D, kFmt, 1, 1>(p, ws, st);
  return rows > 8 ? att_launch<D, kFmt, 2, 2>(p, ws, st) : att_launch<D, kFmt, 1, 2>(p, ws, st);
}

cudaError_t launch_cache_attention(const ckv_cache& c, const ckv_attention_args& a, void* ws, cudaStream_t st) {
  AttArgs p;
  p.c = c;
  p.a = a;
  p.block_log2 = 0;
  while ((1 << p.block_log2) < c.block_size) ++p.block_log2;
  p.group = a.q_heads / c.num_kv_heads;
  p.ctas = kAttMaxCtas;
  p.inv_group = 1.f / p.group;
  p.dense = c.k_tok_stride == c.head_dim && c.v_tok_stride == c.head_dim;
  const int rows = a.max_q * p.group;
  const bool e4 = c.format == CKV_CACHE_E4M3;
  if (c.head_dim == 64)
    return e4 ? att_pick<64, CKV_CACHE_E4M3>(p, rows, ws, st) : att_pick<64, CKV_CACHE_INT8>(p, rows, ws, st);
  return e4 ? att_pick<128, CKV_CACHE_E4M3>(p, rows, ws, st) : att_pick<128, CKV_CACHE_INT8>(p, rows, ws, st);
}

}  // namespace ckv
