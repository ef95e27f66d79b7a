// ce_kv4_decode_attn_score: decode attention and H2O scores over 4-bit pages
// (the format of ce_kv4.cuh).
//
// The batch is split as for bf16 pages (ce_decode.cu): equal contiguous ranges
// of stages per CTA, one partial record (m, l, O) per sequence a CTA touched,
// merged by a combine kernel.  With k = m_k + c_k s_k and v = m_v + c_v s_v per
// token,
//
//   q . k    = s_k (q . c_k) + m_k sum_d q_d
//   sum p v  = sum_t (p_t s_t) c_t  +  (sum_t p_t m_t)
//
// so both matrix products run on the codes themselves and the scales touch
// one value per (token, head) instead of 64.  A code needs no conversion: 4
// bits in the low mantissa bits of an fp16 are the subnormal number c * 2^-24
// (c * 2^-20 for the upper nibble of a byte), which the tensor cores multiply
// exactly.  One 32-bit word of codes is a whole m16n8k16 A fragment of V, or
// two K-steps' halves of K, for four ANDs and a shift.  The other operand
// brings the range back: the query row is scaled by a power of two to
// 2^14 .. 2^15 (1/16 of that where it meets upper nibbles), and a head's weights
// p_t s_t by a power of two, 2^lift, that puts the largest of them so far at
// 2^7 or above and below 2^16, so both are ordinary fp16 numbers.  (The lift
// goes by p_t s_t, not by the scales alone: a row of large values that a head
// does not look at must not push the others out of fp16.)  Rounding p_t s_t to
// fp16 costs at most 2^-11 of it, or 2^-32 of the largest where it falls below
// fp16's normal range; logits, maxima, sums and accumulators are fp32.
//
// A producer warp copies whole pages (all KV heads) into a ring of shared-memory
// stages with untiled bulk copies; the format puts a page's fragments in lane
// order, 16 bytes per lane and operand.  (Loading them from global memory
// straight into registers a stage ahead needed 1.5 times the instructions per
// page and left too few bytes in flight: 178 us instead of 102 for 409 MB.)
//
// Device times.  64 rows of 2K-32K tokens, 8 KV heads (409 MB): 98 us without
// scores (155 instructions per page and head, 58 % of the issue slots; the loads
// alone take 80, 5.1 TB/s), 128 us with sum, max and no scores mixed (max scores
// write and read 4 KB of log-masses per page), 1 KV head (51 MB, copies of 576
// bytes by one warp): 34 us without scores, 45 with max scores.  Outputs of that
// batch are 1.7e-4 (relative norm) from the same pages' in 64 bits, before their
// rounding to bf16.
#include <algorithm>

#include "ce_decode.cuh"
#include "ce_kv4.cuh"

namespace ce {
namespace kv4 {

using decode::GROUP;
using decode::LOG2E;
using decode::LN2;
using decode::Params;

constexpr int NW = 8;                                // consumer warps
constexpr int THREADS = (NW + 1) * 32;               // and one producer warp
constexpr int PPW = 2;                               // pages that a warp computes at a time
constexpr int CTAS_PER_SM = 2;
constexpr int MIN_STAGES_LOG2 = 0;                   // every CTA below min(stages, grid) has one

// Floats of a record: the means of V [H][64], then (maximum, sum of p) [H].
__host__ __device__ constexpr int rec_floats(int H) { return H * (D + 2); }
static_assert(rec_floats(NW * GROUP) <= decode::REC_FLOATS, "the workspace's records hold it");

// D += A(16x16) * B(16x8) in fp16 with fp32 accumulation.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with D = A * B.
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// (lo, hi) as fp16x2, lo in the low half.
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float pow2_bits(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }
constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;

// A warp's running state over one sequence: KV head g's eight query heads,
// this lane's columns being heads 2t and 2t + 1 (lane = 4 r + t) and its
// rows tokens 2r and 2r + 1 of a page (S^T), dims r and r + 8 of a block (O^T).
struct Rows {
  uint32_t qb[4][2];    // B operand of S^T: query codes' partners, fp16
  float qs0, qs1;       // 2^-24 sum of the scaled query row
  float scale;          // sm_scale in log2 units
  float o[4][4];        // sums of w s c 2^-24 (rows r), of w s 16 c 2^-24 (rows r + 8)
  float z0, z1;         // this lane's sums of w m
  // pairs, of head 2t and head 2t + 1, the same in a head's lanes:
  uint64_t kq;          // a power of two: u kq is the logit in log2 units, u = scale (s (q . c) + m sum q)
  uint64_t nm;          // minus a recent maximum of the logits, rounded up to an integer (NO_MAX: none yet)
  uint64_t f;           // 2^lift: w = p 2^lift, p = 2^(u kq - m); every w s so far is below 2^16
  uint64_t l;           // this lane's sums of p
  __nv_bfloat162 bound; // V scales and magnitudes of minima up to here are taken with p up to 2^ROOM_P
};

constexpr float NO_MAX = -3.402823466e38f;   // no logit is below, but for -inf
// log2 of what w s may reach, of how far p may pass 1 and a scale the one that
// the lift was chosen by before it is chosen again, and of what 2^lift may reach
// (w stays far from fp32's end).
constexpr int TOP = 15, ROOM_P = 3, ROOM_S = 4, MAX_LIFT = 105;
// A row of one value has scale 0: 2^OF_MIN of its minimum counts as its scale, so that
// w m stays below 2^76.  (A scale that is not 0 is at least 2^-12 of the minimum.)
constexpr int OF_MIN = -60;

// The bound that goes with the larger of a lane's two lifts.
__device__ __forceinline__ __nv_bfloat162 bound_of(float lift) {
  const int e = 127 + TOP - ROOM_P - static_cast<int>(lift);
  const uint32_t b = static_cast<uint32_t>(min(e, 254) << 7 | min(e - OF_MIN, 254) << 23);
  return *reinterpret_cast<const __nv_bfloat162*>(&b);
}

__device__ __forceinline__ void clear(Rows& s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s.o[i][0] = s.o[i][1] = s.o[i][2] = s.o[i][3] = 0.f;
  s.nm = pair(-NO_MAX, -NO_MAX);
  s.f = pair(pow2_bits(127 + MAX_LIFT), pow2_bits(127 + MAX_LIFT));
  s.bound = bound_of(MAX_LIFT);
  s.l = pair(0.f, 0.f);
  s.z0 = s.z1 = 0.f;
}

// The query operand of head g * 8 + r (q: its 64 values).
__device__ __forceinline__ void load_query(Rows& s, const __nv_bfloat16* q, int t, float scale_log2) {
  float x[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(q + 16 * t + 2 * i);
    x[2 * i] = __uint_as_float(w << 16);
    x[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // exponent field of the row's largest magnitude; the row times 2^(14 - e)
  // has it in [2^14, 2^15).  Beside queries from 2^73 on, 2^k of what that power
  // takes away goes into the scale, which meets keys that are small then: into
  // the logits at the end it would pass fp32's end.
  int ex = static_cast<int>(__float_as_uint(top) >> 23), most = ex;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  const int k = max(0, most - 200);
  ex = max(ex, 20 + k);
  const float f = pow2_bits(268 - ex);
  s.scale = scale_log2 * pow2_bits(127 + k);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] *= f;
    sum += x[i];
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const int d = (ks >> 1) * 8 + (ks & 1) * 2;
    s.qb[ks][0] = pack_f16(x[d], x[d + 4]);
    s.qb[ks][1] = pack_f16(x[d + 1] * 0.0625f, x[d + 5] * 0.0625f);
  }
  const float qs = sum * 5.9604644775390625e-8f;               // 2^-24
  const float kq = pow2_bits(ex + 10 - k);                     // 2^24 / (f 2^k)
  s.qs0 = __shfl_sync(0xffffffffu, qs, 8 * t);
  s.qs1 = __shfl_sync(0xffffffffu, qs, 8 * t + 4);
  s.kq = pair(__shfl_sync(0xffffffffu, kq, 8 * t), __shfl_sync(0xffffffffu, kq, 8 * t + 4));
}

// Untiled bulk copy of `bytes` (a multiple of 16) into shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

struct Side {           // where a scored sequence's page data goes
  int64_t cpos;         // CSR position of the warp's first page
  int64_t capacity;
  int H, hcol;          // this lane's first head
  float *ul, *tl;
};

__device__ __forceinline__ __nv_bfloat162 magnitudes(uint32_t par) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(&par)); }

constexpr float REST = TOP - ROOM_P - ROOM_S;

// log2 of a power of two.
__device__ __forceinline__ int log2_of(float pow2) { return static_cast<int>(__float_as_uint(pow2) >> 23) - 127; }
// What counts as a token's scale.
__device__ __forceinline__ float reach(float scale, float minimum) {
  return fmaxf(scale, fabsf(minimum) * pow2_bits(127 + OF_MIN));
}

// The running state moved so that the maxima cover x0 kq and x1 kq (this lane's
// largest logits) and every w s of the tile (logits u kq, V parameters vp) is at
// most 2^REST.
__device__ __forceinline__ void move(Rows& s, const float (&u)[PPW][4], const uint2 (&vp)[PPW], float x0, float x1) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
  }
  float kq0, kq1, m0, m1, f0, f1, l0, l1;
  split(s.kq, kq0, kq1);
  x0 *= kq0;
  x1 *= kq1;
  split(s.nm, m0, m1);
  split(s.f, f0, f1);
  split(s.l, l0, l1);
  m0 = -m0;
  m1 = -m1;
  const float n0 = fmaxf(m0, ceilf(x0)), n1 = fmaxf(m1, ceilf(x1));
  const float lift0 = log2_of(f0), lift1 = log2_of(f1);
  float r0 = -INFINITY, r1 = -INFINITY;   // log2 of the tile's largest p s
#pragma unroll
  for (int i = 0; i < 2 * PPW; ++i) {
    const uint32_t par = i & 1 ? vp[i / 2].y : vp[i / 2].x;
    const float e = __log2f(reach(__uint_as_float(par << 16), __uint_as_float(par & 0xffff0000u)));
    r0 = fmaxf(r0, u[i / 2][2 * (i & 1)] * kq0 - n0 + e);
    r1 = fmaxf(r1, u[i / 2][2 * (i & 1) + 1] * kq1 - n1 + e);
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, o));
    r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, o));
  }
  // What was added before is below 2^(TOP + m - n) now; the lift may rise again by as much.
  const float t0 = fminf(fminf(lift0 + (n0 - m0), static_cast<float>(MAX_LIFT)), floorf(REST - r0));
  const float t1 = fminf(fminf(lift1 + (n1 - m1), static_cast<float>(MAX_LIFT)), floorf(REST - r1));
  // Sums of p go by 2^(m - n), sums of w by 2^(m - n + change of the lift), which
  // may be further from 1 than an fp32 is though the product is not: in steps.
  s.l = pair(l0 * fast_exp2(m0 - n0), l1 * fast_exp2(m1 - n1));
  float d0 = fmaxf(m0 - n0 + (t0 - lift0), -300.f), d1 = fmaxf(m1 - n1 + (t1 - lift1), -300.f);
  s.nm = pair(-n0, -n1);
  s.f = pair(pow2_bits(127 + static_cast<int>(t0)), pow2_bits(127 + static_cast<int>(t1)));   // t in MAX_LIFT .. REST - 126
  s.bound = bound_of(fmaxf(t0, t1));
#pragma unroll 1
  do {
    const float a0 = fast_exp2(fmaxf(d0, -100.f)), a1 = fast_exp2(fmaxf(d1, -100.f));
    s.z0 *= a0;
    s.z1 *= a1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.o[q][0] *= a0;
      s.o[q][1] *= a1;
      s.o[q][2] *= a0;
      s.o[q][3] *= a1;
    }
    d0 = fminf(d0 + 100.f, 0.f);
    d1 = fminf(d1 + 100.f, 0.f);
  } while (__any_sync(0xffffffffu, d0 < 0.f || d1 < 0.f));
}

// PPW pages (the first `ntok` tokens of them) of KV head g: K slices at kb,
// V slices at vb, one page every `stride` bytes.
template <int stride, bool TAIL, int MODE>
__device__ __forceinline__ void tile(Rows& s, const uint8_t* kb, const uint8_t* vb, int ntok, int lane,
                                     const Side& side) {
  const int r = lane >> 2, t = lane & 3;
  float u[PPW][4];
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    const uint4 w = *reinterpret_cast<const uint4*>(kb + pg * stride + lane * 16);
    uint2 par = *reinterpret_cast<const uint2*>(kb + pg * stride + CODE_BYTES + r * 8);
    const bool va = !TAIL || pg * P + 2 * r < ntok, vb2 = !TAIL || pg * P + 2 * r + 1 < ntok;
    if (!va) par.x = 0u;
    if (!vb2) par.y = 0u;
    float c[4];
    mma_f16_zero(c, w.x & LOW, w.z & LOW, w.x & HIGH, w.z & HIGH, s.qb[0][0], s.qb[0][1]);
    const uint32_t x8 = w.x >> 8, y8 = w.y >> 8, z8 = w.z >> 8, w8 = w.w >> 8;
    mma_f16(c, x8 & LOW, z8 & LOW, x8 & HIGH, z8 & HIGH, s.qb[1][0], s.qb[1][1]);
    mma_f16(c, w.y & LOW, w.w & LOW, w.y & HIGH, w.w & HIGH, s.qb[2][0], s.qb[2][1]);
    mma_f16(c, y8 & LOW, w8 & LOW, y8 & HIGH, w8 & HIGH, s.qb[3][0], s.qb[3][1]);
    // With the scale in s and m, the power of two kq makes exact logits of these:
    // a maximum can be subtracted from them in one step whatever their magnitude.
    const uint64_t by = pair(s.scale, s.scale);
    float sa, ma, sb, mb;
    split(mul2(pair(__uint_as_float(par.x << 16), __uint_as_float(par.x & 0xffff0000u)), by), sa, ma);
    split(mul2(pair(__uint_as_float(par.y << 16), __uint_as_float(par.y & 0xffff0000u)), by), sb, mb);
    u[pg][0] = va ? fmaf(sa, c[0], ma * s.qs0) : -INFINITY;
    u[pg][1] = va ? fmaf(sa, c[1], ma * s.qs1) : -INFINITY;
    u[pg][2] = vb2 ? fmaf(sb, c[2], mb * s.qs0) : -INFINITY;
    u[pg][3] = vb2 ? fmaf(sb, c[3], mb * s.qs1) : -INFINITY;
  }
  // V scales and minima, and what moves the running state: a logit or a scale
  // with which a w s could pass 2^TOP.
  uint2 vp[PPW];
  float x0 = -INFINITY, x1 = -INFINITY;
  __nv_bfloat162 top = s.bound;
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    vp[pg] = *reinterpret_cast<const uint2*>(vb + pg * stride + CODE_BYTES + r * 8);
    if (TAIL && pg * P + 2 * r >= ntok) vp[pg].x = 0u;
    if (TAIL && pg * P + 2 * r + 1 >= ntok) vp[pg].y = 0u;
    top = __hmax2(__hmax2(top, magnitudes(vp[pg].x)), magnitudes(vp[pg].y));
    x0 = max3(x0, u[pg][0], u[pg][2]);
    x1 = max3(x1, u[pg][1], u[pg][3]);
  }
  {
    float a0, a1;
    split(fma2(pair(x0, x1), s.kq, s.nm), a0, a1);
    const bool high = fmaxf(a0, a1) > ROOM_P;
    if (__any_sync(0xffffffffu, high || *reinterpret_cast<const uint32_t*>(&top) != *reinterpret_cast<const uint32_t*>(&s.bound))) {
      // A large scale alone is common where the lift goes by keys of large weight
      // and small values: what counts is its product with the lane's largest weight.
      float f0, f1;
      split(s.f, f0, f1);
      const float ws = fmaxf(a0 + log2_of(f0), a1 + log2_of(f1)) + __log2f(reach(__low2float(top), __high2float(top)));
      if (__any_sync(0xffffffffu, high || ws > TOP))
        move(s, u, vp, x0, x1);
    }
  }
  if (MODE == CE_MODE_MAX) {
    float kq0, kq1;
    split(s.kq, kq0, kq1);
#pragma unroll
    for (int i = 0; i < 2 * PPW; ++i) {
      const int pg = i / 2, h = i & 1, j = 2 * r + h;
      if ((!TAIL || pg * P + j < ntok) && side.cpos + pg < side.capacity)
        *reinterpret_cast<float2*>(side.tl + ((side.cpos + pg) * P + j) * side.H + side.hcol) =
            make_float2(u[pg][2 * h] * kq0, u[pg][2 * h + 1] * kq1);
    }
  }
  uint32_t pt[PPW][2];   // w s in fp16, as B operands of O^T
  float mass[2 * PPW];   // MODE SUM: this lane's share of the pages' masses, heads 2t and 2t + 1
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    float e[4];
    split(fma2(pair(u[pg][0], u[pg][1]), s.kq, s.nm), e[0], e[1]);
    split(fma2(pair(u[pg][2], u[pg][3]), s.kq, s.nm), e[2], e[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = fast_exp2(e[i]);
    const uint64_t both = add2(pair(e[0], e[1]), pair(e[2], e[3]));
    s.l = add2(s.l, both);
    if (MODE == CE_MODE_SUM) split(both, mass[2 * pg], mass[2 * pg + 1]);
    split(mul2(pair(e[0], e[1]), s.f), e[0], e[1]);
    split(mul2(pair(e[2], e[3]), s.f), e[2], e[3]);
    const float sa = __uint_as_float(vp[pg].x << 16), ma = __uint_as_float(vp[pg].x & 0xffff0000u);
    const float sb = __uint_as_float(vp[pg].y << 16), mb = __uint_as_float(vp[pg].y & 0xffff0000u);
    s.z0 = fmaf(e[0], ma, fmaf(e[2], mb, s.z0));
    s.z1 = fmaf(e[1], ma, fmaf(e[3], mb, s.z1));
    pt[pg][0] = movmatrix_trans(pack_f16(e[0] * sa, e[1] * sa));
    pt[pg][1] = movmatrix_trans(pack_f16(e[2] * sb, e[3] * sb));
  }
  // The tensor cores cut what they add to 24 bits of the largest term, always
  // towards 0, which over thousands of positive terms is a drift: they add up
  // one tile's, and the tiles are added in fp32.
  uint4 wv[PPW];
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) wv[pg] = *reinterpret_cast<const uint4*>(vb + pg * stride + (t * 8 + r) * 16);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float c[4];
#pragma unroll
    for (int pg = 0; pg < PPW; ++pg) {
      const uint32_t w = q == 0 ? wv[pg].x : q == 1 ? wv[pg].y : q == 2 ? wv[pg].z : wv[pg].w;
      const uint32_t odd = w >> 8;
      if (pg == 0) mma_f16_zero(c, w & LOW, w & HIGH, odd & LOW, odd & HIGH, pt[pg][0], pt[pg][1]);
      else mma_f16(c, w & LOW, w & HIGH, odd & LOW, odd & HIGH, pt[pg][0], pt[pg][1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s.o[q][i] += c[i];
  }
  if (MODE == CE_MODE_SUM) {
    // Sum the 4 (page, head) shares over the lanes of equal t; each step halves
    // what a lane still carries, and lanes (r, t) of equal r / 2 end with page
    // r / 4, head 2t + r / 2 % 2, whose log2 mass they keep.
    static_assert(PPW == 2, "four shares over eight lanes");
    float h2[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float mine = (r & 4) ? mass[2 + i] : mass[i], yours = (r & 4) ? mass[i] : mass[2 + i];
      h2[i] = mine + __shfl_xor_sync(0xffffffffu, yours, 16);
    }
    const float mine = (r & 2) ? h2[1] : h2[0], yours = (r & 2) ? h2[0] : h2[1];
    float y = mine + __shfl_xor_sync(0xffffffffu, yours, 8);
    y += __shfl_xor_sync(0xffffffffu, y, 4);
    const int pg = r >> 2, h = (r >> 1) & 1;
    if (!(r & 1) && (!TAIL || pg * P < ntok) && side.cpos + pg < side.capacity) {
      float n0, n1;
      split(s.nm, n0, n1);
      side.ul[(side.cpos + pg) * side.H + side.hcol + h] = y > 0.f ? __log2f(y) - (h ? n1 : n0) : -INFINITY;
    }
  }
}

// A warp's WT tokens of a stage, of which `mine` are left in the sequence.
template <int WT, int stride, int MODE>
__device__ __forceinline__ void stage(Rows& s, const uint8_t* kb, const uint8_t* vb, int mine, int lane, Side side) {
  constexpr int STEP = PPW * P;
  if (mine >= WT) {
#pragma unroll 1
    for (int i = 0; i < WT / STEP; ++i) {
      tile<stride, false, MODE>(s, kb + i * PPW * stride, vb + i * PPW * stride, STEP, lane, side);
      side.cpos += PPW;
    }
    return;
  }
#pragma unroll 1
  for (; mine > 0; mine -= STEP) {
    tile<stride, true, MODE>(s, kb, vb, mine, lane, side);
    kb += PPW * stride;
    vb += PPW * stride;
    side.cpos += PPW;
  }
}

// The warp's sums of p over its lanes and the means of V that its weights make
// (which no range of values takes beyond fp32, as sums could be), into rows
// h0 .. h0 + 7 of a record-shaped buffer of H heads.
__device__ __forceinline__ void put(Rows& s, float* rec, int H, int h0, int lane) {
  const int r = lane >> 2, t = lane & 3;
  float l0, l1, m0, m1, f0, f1;
  split(s.l, l0, l1);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    s.z0 += __shfl_xor_sync(0xffffffffu, s.z0, o);
    s.z1 += __shfl_xor_sync(0xffffffffu, s.z1, o);
  }
  split(s.nm, m0, m1);
  split(s.f, f0, f1);
  const float down0 = pow2_bits(127 - log2_of(f0)), down1 = pow2_bits(127 - log2_of(f1));
  const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
  float* o = rec + (h0 + 2 * t) * D + r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    o[q * 16] = fmaf(s.o[q][0], 16777216.f, s.z0) * i0 * down0;
    o[D + q * 16] = fmaf(s.o[q][1], 16777216.f, s.z1) * i1 * down1;
    o[q * 16 + 8] = fmaf(s.o[q][2], 1048576.f, s.z0) * i0 * down0;
    o[D + q * 16 + 8] = fmaf(s.o[q][3], 1048576.f, s.z1) * i1 * down1;
  }
  if (r == 0) {
    float* ml = rec + H * D + (h0 + 2 * t) * 2;
    ml[0] = l0 == 0.f ? -INFINITY : -m0;
    ml[1] = l0;
    ml[2] = l1 == 0.f ? -INFINITY : -m1;
    ml[3] = l1;
  }
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory"); }

// The CTA's record of a sequence.  Below 8 KV heads several warps share a head:
// their parts are merged in shared memory, so that a record has one row per
// head whatever the split.
template <int G>
__device__ __forceinline__ void leave(const Params& p, Rows& s, int b, int warp, int lane, float* part) {
  constexpr int H = G * GROUP, SUB = NW / G;
  float* rec = p.rec + static_cast<int64_t>(b + blockIdx.x) * rec_floats(H);
  if constexpr (SUB == 1) {
    put(s, rec, H, warp * GROUP, lane);
    return;
  }
  consumers_sync();   // the buffer is free (all warps leave the same sequences in the same order)
  put(s, part + (warp / G) * rec_floats(H), H, (warp % G) * GROUP, lane);
  consumers_sync();
  for (int i = threadIdx.x; i < H * D / 2; i += NW * 32) {
    const int h = i / (D / 2);
    float w[SUB], top = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      w[k] = part[k * rec_floats(H) + H * D + 2 * h];
      top = fmaxf(top, w[k]);
    }
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      w[k] = w[k] == -INFINITY ? 0.f : fast_exp2(w[k] - top);
      w[k] *= part[k * rec_floats(H) + H * D + 2 * h + 1];
      l += w[k];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float2 o = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      const float2 x = reinterpret_cast<const float2*>(part + k * rec_floats(H))[i];
      o.x = fmaf(w[k] * inv, x.x, o.x);
      o.y = fmaf(w[k] * inv, x.y, o.y);
    }
    reinterpret_cast<float2*>(rec)[i] = o;
    if (i % (D / 2) == 0) {
      rec[H * D + 2 * h] = top;
      rec[H * D + 2 * h + 1] = l;
    }
  }
}

// Sizes that go with G KV heads: a stage is WT tokens of every consumer warp.
// Below 8 heads several warps share a head and leave() needs a buffer, so
// stages are halved there to keep two CTAs on an SM.
template <int G>
struct Shape {
  static constexpr int H = G * GROUP, SUB = NW / G;
  static constexpr int WT = (SUB == 1 ? 4 : 2) * P;
  static constexpr int ST = WT * SUB, UPS = ST / P;
  static constexpr int UNIT_BYTES = G * SLICE;
  static constexpr int HALF_STAGE = UPS * UNIT_BYTES, STAGE_BYTES = 2 * HALF_STAGE;   // K, then V
  static constexpr int NSTAGES = SUB == 1 ? 3 : 5;
  static constexpr int SMEM = NSTAGES * STAGE_BYTES + (SUB == 1 ? 0 : SUB * rec_floats(H) * 4);
  static_assert(CTAS_PER_SM * (SMEM + 2048) <= 228 * 1024, "two CTAs per SM");
};

template <int M>
struct Mode {
  static constexpr int value = M;
};
struct Ring {   // a consumer's place in the stage ring
  int slot;
  uint32_t phase;
  bool aborted;
};

__device__ __forceinline__ int stages_of(const Params& p, int b, int ST) {
  return (decode::seq_tokens(p, b, P) + ST - 1) / ST;
}

// Warps 0..7 consume (warp w: KV head w % G, every (8 / G)-th group of pages
// of each stage), warp 8 produces.
template <int G>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM)
    attn_kernel(const Params p, const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool) {
  using C = Shape<G>;
  constexpr int H = C::H, WT = C::WT, ST = C::ST, UPS = C::UPS, UNIT_BYTES = C::UNIT_BYTES;
  constexpr int NSTAGES = C::NSTAGES, STAGE_BYTES = C::STAGE_BYTES, HALF_STAGE = C::HALF_STAGE;
  extern __shared__ __align__(128) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem + NSTAGES * STAGE_BYTES);   // leave()
  __shared__ uint64_t full[NSTAGES], empty[NSTAGES];
  __shared__ int64_t scan_sh[32];
  __shared__ int start_sh[2], abort_sh;
  volatile int* abort_flag = &abort_sh;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  launch_dependents();   // the combine launch: its blocks start as this one's leave
  if (tid == 0) {
    for (int s = 0; s < NSTAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], NW);
    }
    *abort_flag = 0;
    start_sh[0] = p.bs;
    start_sh[1] = 0;
    fence_mbar_init();
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");

  // ---- this CTA's range of the batch's stages ---------------------------------
  const int bs = p.bs;
  const int per = (bs + THREADS - 1) / THREADS;
  const int lo_b = min(bs, tid * per), hi_b = min(bs, lo_b + per);
  int64_t local = 0;
  for (int b = lo_b; b < hi_b; ++b) local += stages_of(p, b, ST);
  int64_t S = 0;
  const int64_t excl = decode::block_excl_scan(local, scan_sh, S);   // a barrier: start_sh is set
  const int64_t k = blockIdx.x, grid = decode::eff_grid(S, gridDim.x, MIN_STAGES_LOG2);
  const int S_lo = static_cast<int>(k < grid ? k * S / grid : S);
  const int S_hi = static_cast<int>(k < grid ? (k + 1) * S / grid : S);
  if (S_lo < S_hi && excl <= S_lo && S_lo < excl + local) {
    int64_t run = excl;
    for (int b = lo_b; b < hi_b; ++b) {
      const int n = stages_of(p, b, ST);
      if (S_lo < run + n) {
        start_sh[0] = b;
        start_sh[1] = static_cast<int>(run);
        break;
      }
      run += n;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    int64_t run = excl;
    for (int b = lo_b; b < hi_b; ++b) {
      p.prefix[b] = static_cast<int32_t>(run);
      const int n = stages_of(p, b, ST);
      run += n;
    }
    if (tid == 0) p.prefix[bs] = static_cast<int32_t>(S);
  }

  int b = start_sh[0], base = start_sh[1];
  int nst = 0, tok_b = 0;
  int64_t ip_b = 0;
  auto load_seq = [&](int bb) {
    tok_b = decode::seq_tokens(p, bb, P);
    nst = (tok_b + ST - 1) / ST;
    ip_b = p.kv_indptr[bb];
  };
  if (b < bs) load_seq(b);

  if (warp == NW) {
    // -------------------------------- producer --------------------------------
    // Page indices in 32-entry windows, a third one in flight, as for bf16 pages.
    int issued = 0;
    auto fetch = [&](int64_t w0) -> int {
      const int64_t c = w0 + lane;
      return (c >= 0 && c < p.kv_capacity) ? p.kv_indices[c] : -2;
    };
    int64_t w0 = -1;
    int idx_cur = -2, idx_next = -2, idx_ahead = -2;
    for (int x = S_lo; x < S_hi; ++x, ++issued) {
      while (x >= base + nst) {
        base += nst;
        ++b;
        load_seq(b);
      }
      const int j = x - base;
      const int ntok = min(ST, tok_b - j * ST);
      const int nunits = (ntok + P - 1) / P;
      const int64_t c0 = ip_b + static_cast<int64_t>(j) * UPS;
      if (w0 < 0 || c0 < w0 || c0 + nunits > w0 + 64) {
        w0 = c0;
        idx_cur = fetch(w0);
        idx_next = fetch(w0 + 32);
        idx_ahead = fetch(w0 + 64);
      } else if (c0 >= w0 + 32) {
        w0 += 32;
        idx_cur = idx_next;
        idx_next = idx_ahead;
        idx_ahead = fetch(w0 + 64);
      }
      const int s = issued % NSTAGES;
      if (issued >= NSTAGES && !warp_wait_quiet(&empty[s], ((issued / NSTAGES) & 1) ^ 1, p.err, abort_flag, lane)) {
        *abort_flag = 1;
        break;
      }
      const int slot = static_cast<int>(c0 - w0) + lane;
      const int a = __shfl_sync(0xffffffffu, idx_cur, slot & 31);
      const int bn = __shfl_sync(0xffffffffu, idx_next, slot & 31);
      int unit = -1;
      if (lane < nunits) {
        const int v = slot < 32 ? a : bn;
        if (v == -2) {
          flag_error(p.err, CE_EW_CAPACITY);
        } else if (v < 0 || v >= p.pool_units) {
          flag_error(p.err, CE_EW_INDEX);
        } else {
          unit = v;
        }
      }
      const unsigned valid = __ballot_sync(0xffffffffu, unit >= 0);
      if (lane == 0) mbar_arrive_expect_tx(&full[s], __popc(valid) * UNIT_BYTES * 2);
      __syncwarp();
      if (unit >= 0) {
        uint8_t* kd = smem + s * STAGE_BYTES + lane * UNIT_BYTES;
        const int64_t off = static_cast<int64_t>(unit) * UNIT_BYTES;
        bulk_load(kd, k_pool + off, UNIT_BYTES, &full[s]);
        bulk_load(kd + HALF_STAGE, v_pool + off, UNIT_BYTES, &full[s]);
      }
    }
    // Every load issued lands before the CTA may exit.
    if (lane == 0)
      for (int it = max(0, issued - NSTAGES); it < issued; ++it) mbar_wait(&full[it % NSTAGES], (it / NSTAGES) & 1, p.err);
  } else {
    // ------------------------------- consumers -------------------------------
    const int g = warp % G, tb = warp / G;
    const int head = g * GROUP + (lane >> 2);
    const uint8_t* mine0 = smem + tb * (WT / P) * UNIT_BYTES + g * SLICE;
    Rows st;
    Ring ring{0, 0u, false};
    // After a timeout a warp keeps walking (so that leave()'s barriers and the
    // records stay in step) but waits for and computes nothing more.
    auto begin = [&]() -> const uint8_t* {
      if (!ring.aborted && !mbar_wait_quiet(&full[ring.slot], ring.phase, p.err, abort_flag)) {
        *abort_flag = 1;
        ring.aborted = true;
      }
      return mine0 + ring.slot * STAGE_BYTES;
    };
    auto end = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[ring.slot]);   // release orders the reads above
      if (++ring.slot == NSTAGES) {
        ring.slot = 0;
        ring.phase ^= 1u;
      }
    };
    for (int x = S_lo; x < S_hi;) {
      while (x >= base + nst) {
        base += nst;
        ++b;
        load_seq(b);
      }
      clear(st);
      load_query(st, p.q + static_cast<int64_t>(b) * p.q_sb + static_cast<int64_t>(head) * p.q_sh, lane & 3,
                 p.scale_log2);
      int mode = decode::seq_mode(p, b);
      if ((mode == CE_MODE_SUM && !p.ul) || (mode == CE_MODE_MAX && !p.tl)) {
        if (lane == 0 && warp == 0) flag_error(p.err, CE_EW_MODE);
        mode = CE_MODE_NONE;
      }
      Side side{ip_b + static_cast<int64_t>(x - base) * UPS + tb * (WT / P), p.kv_capacity, H,
                g * GROUP + 2 * (lane & 3), p.ul, p.tl};
      const int stop = min(S_hi, base + nst), whole = min(stop, base + tok_b / ST);
      auto whole_stages = [&](auto md) {
        for (; x < whole; ++x) {
          const uint8_t* kb = begin();
          if (!ring.aborted) stage<WT, UNIT_BYTES, decltype(md)::value>(st, kb, kb + HALF_STAGE, WT, lane, side);
          side.cpos += UPS;
          end();
        }
      };
      if (mode == CE_MODE_SUM) whole_stages(Mode<CE_MODE_SUM>{});
      else if (mode == CE_MODE_MAX) whole_stages(Mode<CE_MODE_MAX>{});
      else whole_stages(Mode<CE_MODE_NONE>{});
      if (x < stop) {   // the sequence's last stage
        const int left = tok_b - (x - base) * ST - tb * WT;   // tokens from this warp's first page on
        const uint8_t *kb = begin(), *vb = kb + HALF_STAGE;
        if (!ring.aborted) {
          if (mode == CE_MODE_SUM) stage<WT, UNIT_BYTES, CE_MODE_SUM>(st, kb, vb, left, lane, side);
          else if (mode == CE_MODE_MAX) stage<WT, UNIT_BYTES, CE_MODE_MAX>(st, kb, vb, left, lane, side);
          else stage<WT, UNIT_BYTES, CE_MODE_NONE>(st, kb, vb, left, lane, side);
        }
        end();
        ++x;
      }
      leave<G>(p, st, b, warp, lane, part);
    }
  }
  __syncthreads();
}

// Output, normaliser and log2 normaliser of every (row, head) from its records:
// W warps each merge every W-th group of slots (lane i: slot i's maximum and
// sum; then the slots' output rows, two dims per lane).
constexpr int CB_THREADS = 256;

template <int H, int W>
__global__ void __launch_bounds__(CB_THREADS) combine_kernel(const Params p, int launched) {
  wait_for_prerequisites();
  // The score launch starts under this one where both are small (12.4 -> 11.0 us
  // for a row of 517 tokens, 20.9 -> 19.2 us for one of 29,719); with a batch's
  // many blocks its waiting ones were in the way (121 -> 126 us for 64 rows of
  // 2K-32K tokens).
  if constexpr (W > 1) launch_dependents();
  constexpr int PER = CB_THREADS / 32 / W;   // (row, head) pairs per block
  __shared__ float sh_o[W > 1 ? W : 1][D], sh_ml[W > 1 ? W : 1][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % W;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * PER + warp / W;
  if (item >= static_cast<int64_t>(p.bs) * H) return;   // the whole block when W > 1
  const int b = static_cast<int>(item / H), h = static_cast<int>(item % H);
  const int64_t S = p.prefix[p.bs], pre = p.prefix[b], n = p.prefix[b + 1] - pre;
  const int64_t grid = decode::eff_grid(S, launched, MIN_STAGES_LOG2);
  int k0 = 0, slots = 0;
  if (n > 0) {
    k0 = decode::cta_of_stage(pre, S, grid);
    slots = decode::cta_of_stage(pre + n - 1, S, grid) - k0 + 1;
  }
  const float* rec = p.rec + static_cast<int64_t>(b + k0) * rec_floats(H);
  float m = -INFINITY, l = 0.f;
  float2 o = make_float2(0.f, 0.f);
  constexpr int BATCH = W > 1 ? 8 : 32;   // slots per round
  for (int s0 = sub * BATCH; s0 < slots; s0 += W * BATCH) {
    const int cnt = min(BATCH, slots - s0);
    const float* base = rec + static_cast<int64_t>(s0) * rec_floats(H);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < cnt) ml = *reinterpret_cast<const float2*>(base + static_cast<int64_t>(lane) * rec_floats(H) + H * D + 2 * h);
    float top = ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    top = fmaxf(top, m);
    float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
    w *= ml.y;
    float sum = w;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const float before = l * (m == -INFINITY ? 0.f : exp2f(m - top));
    l = before + sum;
    const float inv = l == 0.f ? 0.f : 1.f / l;   // o stays a mean
    o.x *= before * inv;
    o.y *= before * inv;
    w *= inv;
    m = top;
    for (int i0 = 0; i0 < cnt; i0 += 8) {
      float2 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = make_float2(0.f, 0.f);
        if (i0 + i < cnt)
          v[i] = *reinterpret_cast<const float2*>(base + static_cast<int64_t>(i0 + i) * rec_floats(H) + h * D + 2 * lane);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, (i0 + i) & 31);
        if (i0 + i < cnt) {
          o.x = fmaf(wi, v[i].x, o.x);
          o.y = fmaf(wi, v[i].y, o.y);
        }
      }
    }
  }
  if constexpr (W > 1) {
    reinterpret_cast<float2*>(sh_o[warp])[lane] = o;
    if (lane == 0) {
      sh_ml[warp][0] = m;
      sh_ml[warp][1] = l;
    }
    __syncthreads();
    if (warp > 0) return;
    m = -INFINITY;
#pragma unroll
    for (int k = 0; k < W; ++k) m = fmaxf(m, sh_ml[k][0]);
    float w[W];
    l = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      w[k] = sh_ml[k][0] == -INFINITY ? 0.f : exp2f(sh_ml[k][0] - m);
      w[k] *= sh_ml[k][1];
      l += w[k];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    o = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 x = reinterpret_cast<const float2*>(sh_o[k])[lane];
      o.x = fmaf(w[k] * inv, x.x, o.x);
      o.y = fmaf(w[k] * inv, x.y, o.y);
    }
  }
  // with the sink in the normaliser; a row with neither tokens nor a sink is
  // zeros and -inf
  const float sink2 = p.sinks ? p.sinks[h] * LOG2E : -INFINITY;
  const float top = fmaxf(m, sink2);
  float L = -INFINITY, f = 0.f;
  if (n > 0 || sink2 != -INFINITY) {
    const float a = l * (m == -INFINITY ? (l != l ? l : 0.f) : exp2f(m - top));   // a row of NaN logits has no maximum
    const float den = a + (p.sinks ? exp2f(sink2 - top) : 0.f);
    L = top + log2f(den);
    f = a / den;
  }
  const int64_t at = static_cast<int64_t>(b) * p.o_sb + static_cast<int64_t>(h) * p.o_sh + 2 * lane;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + at;
  out[0] = __float2bfloat16_rn(n > 0 ? o.x * f : 0.f);
  out[1] = __float2bfloat16_rn(n > 0 ? o.y * f : 0.f);
  if (lane == 0) {
    p.lse2[item] = L;
    if (p.lse_out) p.lse_out[item] = L * LN2;
  }
}

// Page scores of the batch from the combine kernel's normalisers: scores[g, unit]
// += SUM: sum_h 2^(page log-mass - L_h), MAX: sum_t 2^(max_h (s_t,h - L_h)).  Every
// warp takes SC_PAGES consecutive positions of the CSR, all KV heads at once,
// whatever rows they belong to: neighbouring lanes read neighbouring heads,
// and a long row's pages are spread as evenly as the others'.
constexpr int SC_THREADS = 256;
constexpr int SC_PAGES = 4;

template <int G>
__global__ void __launch_bounds__(SC_THREADS) score_kernel(const Params p) {
  constexpr int H = G * GROUP;
  static_assert(SC_PAGES * 8 <= 32, "a lane per (page, head)");
  // lanes as token lanes x heads: TPL tokens each (at G = 1 the upper 16 lanes
  // repeat the lower)
  constexpr int LANES = 32 / G, TL = LANES < P ? LANES : P, TPL = P / TL;
  const int lane = threadIdx.x & 31, g = lane % G, tl = (lane / G) % TL;
  const int64_t end = min(static_cast<int64_t>(p.kv_indptr[p.bs]), p.kv_capacity);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (SC_THREADS / 32) * SC_PAGES;
  float* sc = p.scores + g * p.score_sg;
  bool waited = false;
  for (int64_t c0 = (static_cast<int64_t>(blockIdx.x) * (SC_THREADS / 32) + (threadIdx.x >> 5)) * SC_PAGES; c0 < end;
       c0 += step) {
    // The row of position c0, by 32-way search: kv_indptr[lo] <= c0 < kv_indptr[hi].
    int lo = 0, hi = p.bs;
    while (hi - lo > 1) {
      const int part = (hi - lo + 31) / 32, at = lo + lane * part;
      const unsigned below = __ballot_sync(0xffffffffu, at < hi && p.kv_indptr[at] <= c0);
      const int last = max(0, 31 - __clz(static_cast<int>(below)));   // lane 0's holds unless c0 precedes the list
      hi = min(hi, lo + (last + 1) * part);
      lo += last * part;
    }
    // Lane i < SC_PAGES: the row of position c0 + i, the page's place in it,
    // its valid tokens (0: nothing to score) and unit.
    int row = lo, valid = 0, unit = -1;
    bool fresh = false, sum = false;
    if (lane < SC_PAGES && c0 + lane < end) {
      const int c = static_cast<int>(c0) + lane;
      unit = p.kv_indices[c];
      while (row + 1 < p.bs && p.kv_indptr[row + 1] <= c) ++row;
      const int start = p.kv_indptr[row], tokens = decode::seq_tokens(p, row, P), mode = decode::seq_mode(p, row);
      const int j = c - start;
      sum = mode == CE_MODE_SUM && p.ul;
      // a unit outside the pool was flagged by the attention kernel
      if (j >= 0 && unit >= 0 && unit < p.pool_units && (sum || (mode == CE_MODE_MAX && p.tl))) {
        valid = max(0, min(P, tokens - j * P));
        fresh = p.zero_new && j * P + 1 == tokens;
      }
    }
    // the lists were there before this call; the masses and normalisers come from
    // the two launches before
    if (!waited) wait_for_prerequisites();
    waited = true;
    // SUM pages, one lane per (page, head)
    {
      const int i = min(lane / G, SC_PAGES - 1);
      const int n = __shfl_sync(0xffffffffu, valid, i), b = __shfl_sync(0xffffffffu, row, i);
      const int to = __shfl_sync(0xffffffffu, unit, i);
      const bool is_sum = __shfl_sync(0xffffffffu, sum, i), first = __shfl_sync(0xffffffffu, fresh, i);
      if (n > 0 && is_sum && lane < SC_PAGES * G) {
        const float old = sc[to];
        const float4* l4 = reinterpret_cast<const float4*>(p.lse2 + static_cast<int64_t>(b) * H + g * GROUP);
        const float4* u4 = reinterpret_cast<const float4*>(p.ul + (c0 + i) * H + g * GROUP);
        const float4 L = l4[0], M = l4[1], x = u4[0], y = u4[1];
        const float mass =
            ((fast_exp2(x.x - L.x) + fast_exp2(x.y - L.y)) + (fast_exp2(x.z - L.z) + fast_exp2(x.w - L.w))) +
            ((fast_exp2(y.x - M.x) + fast_exp2(y.y - M.y)) + (fast_exp2(y.z - M.z) + fast_exp2(y.w - M.w)));
        sc[to] = first ? mass : old + mass;
      }
    }
    // MAX pages one after another, their tokens over the lanes
    unsigned todo = __ballot_sync(0xffffffffu, valid > 0 && !sum);
    while (todo) {
      const int i = __ffs(static_cast<int>(todo)) - 1;
      todo &= todo - 1;
      const int n = __shfl_sync(0xffffffffu, valid, i), b = __shfl_sync(0xffffffffu, row, i);
      const int to = __shfl_sync(0xffffffffu, unit, i);
      const bool first = __shfl_sync(0xffffffffu, fresh, i);
      const float4* l4 = reinterpret_cast<const float4*>(p.lse2 + static_cast<int64_t>(b) * H + g * GROUP);
      const float4 L = l4[0], M = l4[1];
      const float old = lane < G ? sc[to] : 0.f;
      float4 x[TPL], y[TPL];
#pragma unroll
      for (int k = 0; k < TPL; ++k) {
        const int t = min(tl + k * TL, n - 1);   // valid tokens only
        const float4* u4 = reinterpret_cast<const float4*>(p.tl + ((c0 + i) * P + t) * H + g * GROUP);
        x[k] = u4[0];
        y[k] = u4[1];
      }
      float mass = 0.f;
#pragma unroll
      for (int k = 0; k < TPL; ++k) {
        const float top =
            fmaxf(fmaxf(fmaxf(x[k].x - L.x, x[k].y - L.y), fmaxf(x[k].z - L.z, x[k].w - L.w)),
                  fmaxf(fmaxf(y[k].x - M.x, y[k].y - M.y), fmaxf(y[k].z - M.z, y[k].w - M.w)));
        mass += tl + k * TL < n ? fast_exp2(top) : 0.f;
      }
#pragma unroll
      for (int o = G; o < G * TL; o <<= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
      if (lane < G) sc[to] = first ? mass : old + mass;
    }
  }
  if (!waited) wait_for_prerequisites();   // so that what follows this launch follows those
}

template <int G>
int launch(const Params& p, const uint8_t* k_pool, const uint8_t* v_pool, int sms, int score_flags, cudaStream_t st) {
  constexpr int H = G * GROUP;
  const int grid = CTAS_PER_SM * sms;
  if (!host::set_smem(attn_kernel<G>, Shape<G>::SMEM)) return host::fail(CE_ERR_CUDA, "smem attr");
  attn_kernel<G><<<grid, THREADS, Shape<G>::SMEM, st>>>(p, k_pool, v_pool);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_decode launch");
  // Few (row, head) pairs have many records each (a row spans many CTAs): a
  // block per pair; many pairs a warp each.
  const int64_t pairs = static_cast<int64_t>(p.bs) * H;
  if (pairs <= 8LL * sms)
    host::launch_after(combine_kernel<H, 8>, static_cast<unsigned>(pairs), CB_THREADS, st, p, grid);
  else
    host::launch_after(combine_kernel<H, 1>, static_cast<unsigned>((pairs + 7) / 8), CB_THREADS, st, p, grid);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_decode combine launch");
  if ((score_flags & CE_SCORE_DEFER) || !(score_flags & 3) || !p.mode_of_row) return CE_OK;
  // The scores are a launch of their own over all pages (a task per row and
  // head, as inside the bf16 combine, left the longest row's pages to one
  // block: 371 us instead of 214 at 64 rows of 2K-32K tokens).
  const int64_t warps = (p.kv_capacity + SC_PAGES - 1) / SC_PAGES;
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((warps + SC_THREADS / 32 - 1) / (SC_THREADS / 32), 16LL * sms));
  host::launch_after(score_kernel<G>, static_cast<unsigned>(blocks), SC_THREADS, st, p);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_decode score launch");
  return CE_OK;
}

template <int G>
int load() {
  cudaFuncAttributes a;
  return host::set_smem(attn_kernel<G>, Shape<G>::SMEM) &&
                 cudaFuncGetAttributes(&a, combine_kernel<G * GROUP, 1>) == cudaSuccess &&
                 cudaFuncGetAttributes(&a, combine_kernel<G * GROUP, 8>) == cudaSuccess &&
                 cudaFuncGetAttributes(&a, score_kernel<G>) == cudaSuccess
             ? CE_OK : CE_ERR_CUDA;
}

}  // namespace kv4
}  // namespace ce

using namespace ce;

namespace {
int check_shape(int32_t bs, int64_t pool_units, int64_t cap, int32_t H, int32_t G, int32_t head_dim, int32_t page_size) {
  if (bs < 0 || pool_units < 0 || cap < 0) return host::fail(CE_ERR_ARG, "ce_kv4_decode: negative size");
  if (head_dim != kv4::D) return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_decode: head_dim must be 64");
  if (G <= 0 || H != kv4::GROUP * G || kv4::NW % G != 0)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_decode: needs 8 query heads per KV head and 1/2/4/8 KV heads");
  if (page_size != kv4::P) return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_decode: page_size must be 16");
  return CE_OK;
}
}  // namespace

extern "C" int64_t ce_kv4_decode_workspace_bytes(int32_t bs, int64_t kv_capacity, int32_t num_q_heads,
                                                 int32_t num_kv_heads, int32_t score_flags) {
  if (bs < 0 || kv_capacity < 0 || num_q_heads <= 0 || num_kv_heads <= 0) return -1;
  const int sms = host::sm_count();
  if (sms <= 0) return -1;
  return static_cast<int64_t>(
      host::decode_layout(bs, kv_capacity, num_q_heads, kv4::P, score_flags, kv4::CTAS_PER_SM * sms).total);
}

extern "C" int ce_kv4_decode_attn_score(const void* q, int64_t q_sb, int64_t q_sh, const void* k_pool,
                                        const void* v_pool, int64_t pool_units, const int32_t* kv_indptr,
                                        const int32_t* kv_indices, const int32_t* kv_tokens, int64_t kv_capacity,
                                        const float* sinks, const int32_t* mode_of_row, const int64_t* rows,
                                        float sm_scale, int32_t bs, int32_t num_q_heads, int32_t num_kv_heads,
                                        int32_t head_dim, int32_t page_size, float* scores, int64_t score_sg,
                                        int32_t zero_new, void* out, int64_t o_sb, int64_t o_sh, float* lse_out,
                                        int32_t score_flags, void* workspace, int64_t workspace_bytes, int32_t* err,
                                        void* stream) {
  const int shape = check_shape(bs, pool_units, kv_capacity, num_q_heads, num_kv_heads, head_dim, page_size);
  if (shape != CE_OK) return shape;
  if (!(sm_scale > 0.f)) return host::fail(CE_ERR_ARG, "ce_kv4_decode: sm_scale must be positive");
  if (bs == 0) return CE_OK;
  if (bs > 65535) return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_decode: more than 65535 rows");
  if (!q || !k_pool || !v_pool || !kv_indptr || !kv_indices || !kv_tokens || !out || !workspace)
    return host::fail(CE_ERR_ARG, "ce_kv4_decode: null pointer");
  if (pool_units == 0) return host::fail(CE_ERR_ARG, "ce_kv4_decode: empty pool");
  if ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return host::fail(CE_ERR_ARG, "ce_kv4_decode: pools and workspace must be 16-byte aligned");
  if ((q_sh | q_sb) & 1 || reinterpret_cast<uintptr_t>(q) & 3)
    return host::fail(CE_ERR_ARG, "ce_kv4_decode: q must be 4-byte aligned with even strides");
  if (mode_of_row && scores && score_sg < pool_units)
    return host::fail(CE_ERR_ARG, "ce_kv4_decode: score head stride below pool_units");
  const int sms = host::sm_count();
  if (sms <= 0) return host::fail(CE_ERR_CUDA, "no device");
  const int grid = kv4::CTAS_PER_SM * sms;
  const host::DecodeLayout L = host::decode_layout(bs, kv_capacity, num_q_heads, kv4::P, score_flags, grid);
  if (workspace_bytes < static_cast<int64_t>(L.total))
    return host::fail(CE_ERR_WORKSPACE, "ce_kv4_decode: workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  decode::Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_sb;
  p.q_sh = q_sh;
  p.kv_indptr = kv_indptr;
  p.kv_indices = kv_indices;
  p.kv_tokens = kv_tokens;
  p.kv_capacity = kv_capacity;
  p.pool_units = pool_units;
  p.sinks = sinks;
  p.mode_of_row = scores ? mode_of_row : nullptr;
  p.rows = rows;
  p.scale_log2 = sm_scale * decode::LOG2E;
  p.bs = bs;
  p.H = num_q_heads;
  p.G = num_kv_heads;
  p.scores = scores;
  p.score_sg = score_sg;
  p.zero_new = zero_new;
  p.out = out;
  p.o_sb = o_sb;
  p.o_sh = o_sh;
  p.lse_out = lse_out;
  p.prefix = reinterpret_cast<int32_t*>(ws + L.prefix);
  p.lse2 = reinterpret_cast<float*>(ws + L.lse2);
  p.rec = reinterpret_cast<float*>(ws + L.rec);
  p.ul = (score_flags & 3) ? reinterpret_cast<float*>(ws + L.ul) : nullptr;
  p.tl = (score_flags & 2) ? reinterpret_cast<float*>(ws + L.tl) : nullptr;
  p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t *kp = static_cast<const uint8_t*>(k_pool), *vp = static_cast<const uint8_t*>(v_pool);
  switch (num_kv_heads) {
    case 1: return kv4::launch<1>(p, kp, vp, sms, score_flags, st);
    case 2: return kv4::launch<2>(p, kp, vp, sms, score_flags, st);
    case 4: return kv4::launch<4>(p, kp, vp, sms, score_flags, st);
    default: return kv4::launch<8>(p, kp, vp, sms, score_flags, st);
  }
}

int ce::host::kv4_prepare_device() {
  if (kv4::load<1>() != CE_OK || kv4::load<2>() != CE_OK || kv4::load<4>() != CE_OK || kv4::load<8>() != CE_OK)
    return host::fail_cuda("4-bit decode kernels: set-up");
  return host::kv4_copy_prepare_device();
}
