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
// 2^14 .. 2^15 (1/16 of that where it meets upper nibbles), and the weights
// p_t s_t by 2^15 over a power of two above every scale seen so far, so both
// are ordinary fp16 numbers.  Rounding them to fp16 (2^-12 relative at most,
// 2^-39 of the largest) is far below the output's bf16 rounding; logits,
// maxima, sums and accumulators are fp32.
//
// A producer warp copies whole pages (all KV heads) into a ring of shared-memory
// stages with untiled bulk copies; the format puts a page's fragments in lane
// order, 16 bytes per lane and operand.  (Loading them from global memory
// straight into registers a stage ahead needed 221 instructions per page and
// head instead of 143 and left too few bytes in flight: 178 us instead of 102
// for 409 MB.)
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

// Floats of a record: the unnormalised outputs [H][64], then (maximum, sum) [H].
__host__ __device__ constexpr int rec_floats(int H) { return H * (D + 2); }

// D += A(16x16) * B(16x8) in fp16 with fp32 accumulation.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
  float kq0, kq1;       // log2-domain logit of u = s (q . c) + m sum q
  float o[4][4];
  float m0, m1, l0, l1; // running maxima (shared by the lanes of a head), this lane's sums
  float z0, z1;         // this lane's sum p m
  float bound, inv;     // a power of two above every V scale so far, 2^15 / bound
};

constexpr float MIN_BOUND = 7.888609052210118e-31f;   // 2^-100

__device__ __forceinline__ void clear(Rows& s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s.o[i][0] = s.o[i][1] = s.o[i][2] = s.o[i][3] = 0.f;
  s.m0 = s.m1 = -INFINITY;
  s.l0 = s.l1 = s.z0 = s.z1 = 0.f;
  s.bound = MIN_BOUND;
  s.inv = 32768.f / MIN_BOUND;
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
  // has it in [2^14, 2^15)
  const int ex = max(static_cast<int>(__float_as_uint(top) >> 23), 20);
  const float f = pow2_bits(268 - ex);
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
  const float kq = scale_log2 * pow2_bits(min(ex + 10, 254));  // 2^24 / f
  s.qs0 = __shfl_sync(0xffffffffu, qs, 8 * t);
  s.qs1 = __shfl_sync(0xffffffffu, qs, 8 * t + 4);
  s.kq0 = __shfl_sync(0xffffffffu, kq, 8 * t);
  s.kq1 = __shfl_sync(0xffffffffu, kq, 8 * t + 4);
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
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    mma_f16(c, w.x & LOW, w.z & LOW, w.x & HIGH, w.z & HIGH, s.qb[0][0], s.qb[0][1]);
    mma_f16(c, (w.x >> 8) & LOW, (w.z >> 8) & LOW, (w.x >> 8) & HIGH, (w.z >> 8) & HIGH, s.qb[1][0], s.qb[1][1]);
    mma_f16(c, w.y & LOW, w.w & LOW, w.y & HIGH, w.w & HIGH, s.qb[2][0], s.qb[2][1]);
    mma_f16(c, (w.y >> 8) & LOW, (w.w >> 8) & LOW, (w.y >> 8) & HIGH, (w.w >> 8) & HIGH, s.qb[3][0], s.qb[3][1]);
    const float sa = __uint_as_float(par.x << 16), ma = __uint_as_float(par.x & 0xffff0000u);
    const float sb = __uint_as_float(par.y << 16), mb = __uint_as_float(par.y & 0xffff0000u);
    u[pg][0] = va ? fmaf(sa, c[0], ma * s.qs0) : -INFINITY;
    u[pg][1] = va ? fmaf(sa, c[1], ma * s.qs1) : -INFINITY;
    u[pg][2] = vb2 ? fmaf(sb, c[2], mb * s.qs0) : -INFINITY;
    u[pg][3] = vb2 ? fmaf(sb, c[3], mb * s.qs1) : -INFINITY;
  }
  // V scales and minima, and what could move the running state: a logit above
  // its head's maximum, or a V scale at or above the bound.
  uint2 vp[PPW];
  float x0 = fmaxf(u[0][0], u[0][2]), x1 = fmaxf(u[0][1], u[0][3]), top = 0.f;
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    vp[pg] = *reinterpret_cast<const uint2*>(vb + pg * stride + CODE_BYTES + r * 8);
    if (TAIL && pg * P + 2 * r >= ntok) vp[pg].x = 0u;
    if (TAIL && pg * P + 2 * r + 1 >= ntok) vp[pg].y = 0u;
    top = fmaxf(top, fmaxf(__uint_as_float(vp[pg].x << 16), __uint_as_float(vp[pg].y << 16)));
    if (pg == 0) continue;
    x0 = fmaxf(x0, fmaxf(u[pg][0], u[pg][2]));
    x1 = fmaxf(x1, fmaxf(u[pg][1], u[pg][3]));
  }
  if (__any_sync(0xffffffffu, x0 * s.kq0 > s.m0 || x1 * s.kq1 > s.m1 || top >= s.bound)) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const float n0 = fmaxf(s.m0, x0 * s.kq0), n1 = fmaxf(s.m1, x1 * s.kq1);
    const float a0 = n0 == -INFINITY ? 1.f : fast_exp2(s.m0 - n0), a1 = n1 == -INFINITY ? 1.f : fast_exp2(s.m1 - n1);
    s.m0 = n0;
    s.m1 = n1;
    s.l0 *= a0;
    s.l1 *= a1;
    s.z0 *= a0;
    s.z1 *= a1;
    float f = 1.f;
    if (top >= s.bound) {   // the same for every lane
      const float nb = pow2_bits(min(static_cast<int>(__float_as_uint(top) >> 23) + 1, 253));
      f = s.bound * (1.f / nb);
      s.bound = nb;
      s.inv = 32768.f / nb;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.o[q][0] *= a0 * f;
      s.o[q][1] *= a1 * f;
      s.o[q][2] *= a0 * f;
      s.o[q][3] *= a1 * f;
    }
  }
  const float b0 = s.m0 == -INFINITY ? 0.f : s.m0, b1 = s.m1 == -INFINITY ? 0.f : s.m1;
  float mass[2 * PPW];   // MODE SUM: this lane's share of the pages' masses, heads 2t and 2t + 1
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    float e[4];
    e[0] = fast_exp2(fmaf(u[pg][0], s.kq0, -b0));
    e[1] = fast_exp2(fmaf(u[pg][1], s.kq1, -b1));
    e[2] = fast_exp2(fmaf(u[pg][2], s.kq0, -b0));
    e[3] = fast_exp2(fmaf(u[pg][3], s.kq1, -b1));
    mass[2 * pg] = e[0] + e[2];
    mass[2 * pg + 1] = e[1] + e[3];
    s.l0 += mass[2 * pg];
    s.l1 += mass[2 * pg + 1];
    const float sa = __uint_as_float(vp[pg].x << 16) * s.inv, ma = __uint_as_float(vp[pg].x & 0xffff0000u);
    const float sb = __uint_as_float(vp[pg].y << 16) * s.inv, mb = __uint_as_float(vp[pg].y & 0xffff0000u);
    s.z0 = fmaf(e[0], ma, fmaf(e[2], mb, s.z0));
    s.z1 = fmaf(e[1], ma, fmaf(e[3], mb, s.z1));
    const uint32_t p0 = movmatrix_trans(pack_f16(e[0] * sa, e[1] * sa));
    const uint32_t p1 = movmatrix_trans(pack_f16(e[2] * sb, e[3] * sb));
    const uint4 w = *reinterpret_cast<const uint4*>(vb + pg * stride + (t * 8 + r) * 16);
    const uint32_t wq[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q)
      mma_f16(s.o[q], wq[q] & LOW, wq[q] & HIGH, (wq[q] >> 8) & LOW, (wq[q] >> 8) & HIGH, p0, p1);
    if (MODE == CE_MODE_MAX) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 2 * r + h;
        if ((!TAIL || pg * P + j < ntok) && side.cpos + pg < side.capacity)
          *reinterpret_cast<float2*>(side.tl + ((side.cpos + pg) * P + j) * side.H + side.hcol) =
              make_float2(u[pg][2 * h] * s.kq0, u[pg][2 * h + 1] * s.kq1);
      }
    }
  }
  if (MODE == CE_MODE_SUM) {
    // Sum the 4 (page, head) shares over the lanes of equal t; each step halves
    // what a lane still carries, and lanes (r, t) of equal r / 2 end with page
    // r / 4, head 2t + r / 2 % 2, whose log2 mass under the running maximum they keep.
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
    if (!(r & 1) && (!TAIL || pg * P < ntok) && side.cpos + pg < side.capacity)
      side.ul[(side.cpos + pg) * side.H + side.hcol + h] = y > 0.f ? (h ? b1 : b0) + __log2f(y) : -INFINITY;
  }
}

// The warp's sums over its lanes, and its output row in place: head 2t of dims
// 16 q + r (i = 0) and 16 q + r + 8 (i = 2), head 2t + 1 likewise (i = 1, 3).
__device__ __forceinline__ void finish(Rows& s) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    s.l0 += __shfl_xor_sync(0xffffffffu, s.l0, o);
    s.l1 += __shfl_xor_sync(0xffffffffu, s.l1, o);
    s.z0 += __shfl_xor_sync(0xffffffffu, s.z0, o);
    s.z1 += __shfl_xor_sync(0xffffffffu, s.z1, o);
  }
  // accumulators hold sum (p s 2^15 / bound) (c 2^-24), upper nibbles 16-fold;
  // bound 2^9 in two steps that cannot overflow
  const float fb = s.bound * 9.5367431640625e-7f;   // 2^-20
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    s.o[q][0] = fmaf(s.o[q][0] * 536870912.f, fb, s.z0);
    s.o[q][1] = fmaf(s.o[q][1] * 536870912.f, fb, s.z1);
    s.o[q][2] = fmaf(s.o[q][2] * 33554432.f, fb, s.z0);
    s.o[q][3] = fmaf(s.o[q][3] * 33554432.f, fb, s.z1);
  }
}

// A warp's heads into rows h0 .. h0 + 7 of a record-shaped buffer of H heads.
__device__ __forceinline__ void put(const Rows& s, float* rec, int H, int h0, int lane) {
  const int r = lane >> 2, t = lane & 3;
  float* o = rec + (h0 + 2 * t) * D + r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    o[q * 16] = s.o[q][0];
    o[D + q * 16] = s.o[q][1];
    o[q * 16 + 8] = s.o[q][2];
    o[D + q * 16 + 8] = s.o[q][3];
  }
  if (r == 0) {
    float* ml = rec + H * D + (h0 + 2 * t) * 2;
    ml[0] = s.m0;
    ml[1] = s.l0;
    ml[2] = s.m1;
    ml[3] = s.l1;
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
  finish(s);
  if constexpr (SUB == 1) {
    put(s, rec, H, warp * GROUP, lane);
    return;
  }
  consumers_sync();   // the buffer is free (all warps leave the same sequences in the same order)
  put(s, part + (warp / G) * rec_floats(H), H, (warp % G) * GROUP, lane);
  consumers_sync();
  for (int i = threadIdx.x; i < H * D / 2; i += NW * 32) {
    const int h = i / (D / 2);
    float m[SUB], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      m[k] = part[k * rec_floats(H) + H * D + 2 * h];
      top = fmaxf(top, m[k]);
    }
    float2 o = make_float2(0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      const float* q = part + k * rec_floats(H);
      const float w = m[k] == -INFINITY ? 0.f : fast_exp2(m[k] - top);
      const float2 x = reinterpret_cast<const float2*>(q)[i];
      o.x += w * x.x;
      o.y += w * x.y;
      l += w * q[H * D + 2 * h + 1];
    }
    reinterpret_cast<float2*>(rec)[i] = o;
    if (i % (D / 2) == 0) {
      rec[H * D + 2 * h] = top;
      rec[H * D + 2 * h + 1] = l;
    }
  }
}

// The batch's stages in order: sequence b from stage `base` on, its tokens and
// first CSR position; the next sequence's are loaded one sequence ahead.
template <int ST>
struct Cursor {
  int b, base, tok, nst, next_tok;
  int64_t ip, next_ip;
  __device__ __forceinline__ void fetch_next(const Params& p) {
    const bool more = b + 1 < p.bs;
    next_tok = more ? decode::seq_tokens(p, b + 1, P) : 0;
    next_ip = more ? p.kv_indptr[b + 1] : 0;
  }
  __device__ __forceinline__ void start(const Params& p, int bb, int first) {
    b = bb;
    base = first;
    tok = b < p.bs ? decode::seq_tokens(p, b, P) : 0;
    ip = b < p.bs ? p.kv_indptr[b] : 0;
    nst = (tok + ST - 1) / ST;
    fetch_next(p);
  }
  __device__ __forceinline__ void to(const Params& p, int x) {   // x below the batch's stages
    while (x >= base + nst) {
      base += nst;
      ++b;
      tok = next_tok;
      ip = next_ip;
      nst = (tok + ST - 1) / ST;
      fetch_next(p);
    }
  }
};

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
  const int64_t S_lo = k < grid ? k * S / grid : S, S_hi = k < grid ? (k + 1) * S / grid : S;
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
    for (int64_t x = S_lo; x < S_hi; ++x, ++issued) {
      while (x >= base + nst) {
        base += nst;
        ++b;
        load_seq(b);
      }
      const int j = static_cast<int>(x - base);
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
      if (issued >= NSTAGES && !warp_wait(&empty[s], ((issued / NSTAGES) & 1) ^ 1, p.err, abort_flag, lane)) {
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
    Rows st;
    Side side{0, p.kv_capacity, H, g * GROUP + 2 * (lane & 3), p.ul, p.tl};
    int cur_b = -1, mode = CE_MODE_NONE, s = 0;
    uint32_t ph = 0;
    bool aborted = false;
    for (int64_t x = S_lo; x < S_hi; ++x) {
      while (x >= base + nst) {
        base += nst;
        ++b;
        load_seq(b);
      }
      if (b != cur_b) {
        if (cur_b >= 0) leave<G>(p, st, cur_b, warp, lane, part);
        cur_b = b;
        clear(st);
        load_query(st, p.q + static_cast<int64_t>(b) * p.q_sb + static_cast<int64_t>(head) * p.q_sh, lane & 3,
                   p.scale_log2);
        mode = decode::seq_mode(p, b);
        if ((mode == CE_MODE_SUM && !p.ul) || (mode == CE_MODE_MAX && !p.tl)) {
          if (lane == 0 && warp == 0) flag_error(p.err, CE_EW_MODE);
          mode = CE_MODE_NONE;
        }
      }
      const int j = static_cast<int>(x - base);
      const int mine = tok_b - j * ST - tb * WT;   // tokens from this warp's first page on
      const int cs = s;
      const uint32_t cph = ph;
      if (++s == NSTAGES) {
        s = 0;
        ph ^= 1u;
      }
      // After a timeout the warp keeps walking (so the record writes stay in
      // step) but waits for and computes nothing more.
      if (!aborted && !mbar_wait_or_abort(&full[cs], cph, p.err, abort_flag)) {
        *abort_flag = 1;
        aborted = true;
      }
      if (aborted) continue;
      const uint8_t* kb = smem + cs * STAGE_BYTES + tb * (WT / P) * UNIT_BYTES + g * SLICE;
      const uint8_t* vb = kb + HALF_STAGE;
      side.cpos = ip_b + static_cast<int64_t>(j) * UPS + tb * (WT / P);
      constexpr int STEP = PPW * P;
#pragma unroll 1
      for (int left = mine; left > max(mine - WT, 0); left -= STEP) {
        if (left >= STEP) {
          if (mode == CE_MODE_SUM) tile<UNIT_BYTES, false, CE_MODE_SUM>(st, kb, vb, STEP, lane, side);
          else if (mode == CE_MODE_MAX) tile<UNIT_BYTES, false, CE_MODE_MAX>(st, kb, vb, STEP, lane, side);
          else tile<UNIT_BYTES, false, CE_MODE_NONE>(st, kb, vb, STEP, lane, side);
        } else {
          if (mode == CE_MODE_SUM) tile<UNIT_BYTES, true, CE_MODE_SUM>(st, kb, vb, left, lane, side);
          else if (mode == CE_MODE_MAX) tile<UNIT_BYTES, true, CE_MODE_MAX>(st, kb, vb, left, lane, side);
          else tile<UNIT_BYTES, true, CE_MODE_NONE>(st, kb, vb, left, lane, side);
        }
        kb += PPW * UNIT_BYTES;
        vb += PPW * UNIT_BYTES;
        side.cpos += PPW;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[cs]);   // release orders the reads above
    }
    if (cur_b >= 0) leave<G>(p, st, cur_b, warp, lane, part);
  }
  __syncthreads();
}

// Output, normaliser and log2 normaliser of every (row, head) from its records:
// W warps each merge every W-th group of slots (lane i: slot i's maximum and
// sum; then the slots' output rows, two dims per lane).
constexpr int CB_THREADS = 256;

template <int H, int W>
__global__ void __launch_bounds__(CB_THREADS) combine_kernel(const Params p, int launched) {
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
    const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
    float sum = w * ml.y;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const float a = m == -INFINITY ? 0.f : exp2f(m - top);
    l = l * a + sum;
    o.x *= a;
    o.y *= a;
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
    l = 0.f;
    o = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float a = sh_ml[k][0] == -INFINITY ? 0.f : exp2f(sh_ml[k][0] - m);
      const float2 x = reinterpret_cast<const float2*>(sh_o[k])[lane];
      l += a * sh_ml[k][1];
      o.x = fmaf(a, x.x, o.x);
      o.y = fmaf(a, x.y, o.y);
    }
  }
  // with the sink in the normaliser; a row with neither tokens nor a sink is
  // zeros and -inf
  const float sink2 = p.sinks ? p.sinks[h] * LOG2E : -INFINITY;
  const float top = fmaxf(m, sink2);
  float L = -INFINITY, f = 0.f;
  if (n > 0 || sink2 != -INFINITY) {
    const float a = m == -INFINITY ? (l != l ? l : 0.f) : exp2f(m - top);   // a row of NaN logits has no maximum
    const float den = l * a + (p.sinks ? exp2f(sink2 - top) : 0.f);
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
// += SUM: sum_h 2^(page log-mass - L_h), MAX: sum_t 2^(max_h (s_t,h - L_h)).  Block
// (x, b) takes every gridDim.x-th group of pages of row b, all KV heads at
// once, so that neighbouring threads read neighbouring heads and pages.
constexpr int SC_THREADS = 256;

template <int G>
__global__ void __launch_bounds__(SC_THREADS) score_kernel(const Params p) {
  constexpr int H = G * GROUP;
  const int b = blockIdx.y;
  const int mode = decode::seq_mode(p, b);
  if ((mode != CE_MODE_SUM || !p.ul) && (mode != CE_MODE_MAX || !p.tl)) return;
  const int tokens = decode::seq_tokens(p, b, P);
  const int npages = (tokens + P - 1) / P;
  const int64_t ip = p.kv_indptr[b];
  const int fresh = p.zero_new && (tokens - 1) % P == 0 ? npages - 1 : -1;
  const int lane = threadIdx.x & 31;
  const int g = lane % G;
  float L[GROUP];
  {
    const float4* l4 = reinterpret_cast<const float4*>(p.lse2 + static_cast<int64_t>(b) * H + g * GROUP);
    const float4 x = l4[0], y = l4[1];
    L[0] = x.x, L[1] = x.y, L[2] = x.z, L[3] = x.w, L[4] = y.x, L[5] = y.y, L[6] = y.z, L[7] = y.w;
  }
  float* sc = p.scores + g * p.score_sg;
  auto add = [&](int j, float mass) {
    const int unit = p.kv_indices[ip + j];
    if (unit < 0 || unit >= p.pool_units) return;   // flagged by the attention kernel
    sc[unit] = j == fresh ? mass : sc[unit] + mass;
  };
  if (mode == CE_MODE_SUM) {
    constexpr int PB = SC_THREADS / G;   // pages per block and round
    for (int j = blockIdx.x * PB + threadIdx.x / G; j < npages; j += gridDim.x * PB) {
      if (ip + j >= p.kv_capacity) break;
      const float4* u4 = reinterpret_cast<const float4*>(p.ul + (ip + j) * H + g * GROUP);
      const float4 x = u4[0], y = u4[1];
      const float u[GROUP] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      float mass = 0.f;
#pragma unroll
      for (int r = 0; r < GROUP; ++r) mass += fast_exp2(u[r] - L[r]);
      add(j, mass);
    }
    return;
  }
  // A warp's lanes are token lanes x heads: a page takes TL of them (one page
  // per warp, two at G = 1), TPL tokens each.
  constexpr int LANES = 32 / G, TL = LANES < P ? LANES : P, TPL = P / TL, PW = LANES / TL;
  const int tl = (lane / G) % TL, pw = lane / (G * TL);
  const int step = gridDim.x * (SC_THREADS / 32) * PW;
  for (int j0 = (blockIdx.x * (SC_THREADS / 32) + (threadIdx.x >> 5)) * PW; j0 < npages; j0 += step) {
    const int j = j0 + pw;
    const bool in = j < npages && ip + j < p.kv_capacity;
    float mass = 0.f;
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const int t = tl + i * TL;
      if (in && j * P + t < tokens) {
        const float4* u4 = reinterpret_cast<const float4*>(p.tl + ((ip + j) * P + t) * H + g * GROUP);
        const float4 x = u4[0], y = u4[1];
        const float top = fmaxf(fmaxf(fmaxf(x.x - L[0], x.y - L[1]), fmaxf(x.z - L[2], x.w - L[3])),
                                fmaxf(fmaxf(y.x - L[4], y.y - L[5]), fmaxf(y.z - L[6], y.w - L[7])));
        mass += fast_exp2(top);
      }
    }
#pragma unroll
    for (int o = G; o < G * TL; o <<= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    if (in && tl == 0) add(j, mass);
  }
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
    combine_kernel<H, 8><<<static_cast<unsigned>(pairs), CB_THREADS, 0, st>>>(p, grid);
  else
    combine_kernel<H, 1><<<static_cast<unsigned>((pairs + 7) / 8), CB_THREADS, 0, st>>>(p, grid);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_decode combine launch");
  if ((score_flags & CE_SCORE_DEFER) || !(score_flags & 3) || !p.mode_of_row) return CE_OK;
  // The scores are a launch of their own over all pages, about four blocks per
  // SM over the batch (a task per row and head, as inside the bf16 combine,
  // left the longest row's pages to one block: 371 us instead of 214).
  const int x = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((4LL * sms + p.bs - 1) / p.bs, 512)));
  score_kernel<G><<<dim3(x, p.bs), SC_THREADS, 0, st>>>(p);
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
  p.min_log2 = kv4::MIN_STAGES_LOG2;
  p.window = -1;
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
