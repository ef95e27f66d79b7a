// ce_kv4_decode_attn_score: decode attention and H2O scores over 4-bit pages
// (the format of ce_kv4.cuh).
//
// The batch is split, recorded and combined as for bf16 pages (ce_decode.cu):
// equal contiguous ranges of stages per CTA, one partial record (m, l, O) per
// sequence a CTA touched, and the combine kernel over the records.  What is
// new is the tile.  With k = m_k + c_k s_k and v = m_v + c_v s_v per token,
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
#include <algorithm>

#include "ce_decode.cuh"
#include "ce_kv4.cuh"

namespace ce {
namespace kv4 {

using decode::GROUP;
using decode::LOG2E;
using decode::NCW;
using decode::Params;
using decode::REC_FLOATS;
using decode::REC_ROWS;

constexpr int PPW = 4;                               // pages per warp and stage
constexpr int WT = PPW * P;                          // tokens per warp and stage
constexpr int HALF_STAGE = NCW * PPW * SLICE;        // 18 KB of K (or V)
constexpr int STAGE_BYTES = 2 * HALF_STAGE;
constexpr int NSTAGES = 3;
constexpr int NPW = 2;                               // producer warps
constexpr int THREADS = (NCW + NPW) * 32;
constexpr int SMEM_BYTES = NSTAGES * STAGE_BYTES + 512;
constexpr int CTAS_PER_SM = 2;
constexpr int MIN_STAGES_LOG2 = 0;
static_assert(CTAS_PER_SM * (SMEM_BYTES + 1024) <= 228 * 1024, "two CTAs per SM");

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

// Untiled bulk copy of `bytes` (a multiple of 16) into shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
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

struct Side {           // where a scored sequence's page data goes
  int mode;
  int64_t cpos;         // CSR position of the warp's first page
  int64_t capacity;
  int H, hcol;          // this lane's first head
  float *ul, *tl;
};

// PPW pages (the first `ntok` tokens of them) of KV head g: K slices at kb,
// V slices at vb, one page every `stride` bytes.
template <bool TAIL>
__device__ __forceinline__ void tile(Rows& s, const uint8_t* kb, const uint8_t* vb, int stride, int ntok, int lane,
                                     const Side& side) {
  const int r = lane >> 2;
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
  float x0 = fmaxf(u[0][0], u[0][2]), x1 = fmaxf(u[0][1], u[0][3]);
#pragma unroll
  for (int pg = 1; pg < PPW; ++pg) {
    x0 = fmaxf(x0, fmaxf(u[pg][0], u[pg][2]));
    x1 = fmaxf(x1, fmaxf(u[pg][1], u[pg][3]));
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
  }
  const float n0 = fmaxf(s.m0, x0 * s.kq0), n1 = fmaxf(s.m1, x1 * s.kq1);
  const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
  // Rescale the running state only when some head's maximum moved.
  if (__any_sync(0xffffffffu, n0 != s.m0 || n1 != s.m1)) {
    const float a0 = fast_exp2(s.m0 - b0), a1 = fast_exp2(s.m1 - b1);
    s.l0 *= a0;
    s.l1 *= a1;
    s.z0 *= a0;
    s.z1 *= a1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.o[q][0] *= a0;
      s.o[q][1] *= a1;
      s.o[q][2] *= a0;
      s.o[q][3] *= a1;
    }
    s.m0 = n0;
    s.m1 = n1;
  }
  // V scales and minima; the bound grows (rarely) to stay above every scale.
  uint2 vp[PPW];
  float top = 0.f;
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    vp[pg] = *reinterpret_cast<const uint2*>(vb + pg * stride + CODE_BYTES + r * 8);
    if (TAIL && pg * P + 2 * r >= ntok) vp[pg].x = 0u;
    if (TAIL && pg * P + 2 * r + 1 >= ntok) vp[pg].y = 0u;
    top = fmaxf(top, fmaxf(__uint_as_float(vp[pg].x << 16), __uint_as_float(vp[pg].y << 16)));
  }
  if (__any_sync(0xffffffffu, top >= s.bound)) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float nb = pow2_bits(min(static_cast<int>(__float_as_uint(top) >> 23) + 1, 253));
    const float f = s.bound * (1.f / nb);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.o[q][i] *= f;
    s.bound = nb;
    s.inv = 32768.f / nb;
  }
#pragma unroll
  for (int pg = 0; pg < PPW; ++pg) {
    float e[4];
    e[0] = fast_exp2(fmaf(u[pg][0], s.kq0, -b0));
    e[1] = fast_exp2(fmaf(u[pg][1], s.kq1, -b1));
    e[2] = fast_exp2(fmaf(u[pg][2], s.kq0, -b0));
    e[3] = fast_exp2(fmaf(u[pg][3], s.kq1, -b1));
    const float t0 = e[0] + e[2], t1 = e[1] + e[3];
    s.l0 += t0;
    s.l1 += t1;
    const float sa = __uint_as_float(vp[pg].x << 16) * s.inv, ma = __uint_as_float(vp[pg].x & 0xffff0000u);
    const float sb = __uint_as_float(vp[pg].y << 16) * s.inv, mb = __uint_as_float(vp[pg].y & 0xffff0000u);
    s.z0 = fmaf(e[0], ma, fmaf(e[2], mb, s.z0));
    s.z1 = fmaf(e[1], ma, fmaf(e[3], mb, s.z1));
    const uint32_t p0 = movmatrix_trans(pack_f16(e[0] * sa, e[1] * sa));
    const uint32_t p1 = movmatrix_trans(pack_f16(e[2] * sb, e[3] * sb));
    const uint4 w = *reinterpret_cast<const uint4*>(vb + pg * stride + ((lane & 3) * 8 + r) * 16);
    const uint32_t wq[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q)
      mma_f16(s.o[q], wq[q] & LOW, wq[q] & HIGH, (wq[q] >> 8) & LOW, (wq[q] >> 8) & HIGH, p0, p1);
    if (side.mode == CE_MODE_SUM) {
      // log2 of the page's mass under the running maximum
      float y0 = t0, y1 = t1;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        y0 += __shfl_xor_sync(0xffffffffu, y0, o);
        y1 += __shfl_xor_sync(0xffffffffu, y1, o);
      }
      if (r == 0 && (!TAIL || pg * P < ntok) && side.cpos + pg < side.capacity)
        *reinterpret_cast<float2*>(side.ul + (side.cpos + pg) * side.H + side.hcol) =
            make_float2(y0 > 0.f ? b0 + __log2f(y0) : -INFINITY, y1 > 0.f ? b1 + __log2f(y1) : -INFINITY);
    } else if (side.mode == CE_MODE_MAX) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 2 * r + h;
        if ((!TAIL || pg * P + j < ntok) && side.cpos + pg < side.capacity)
          *reinterpret_cast<float2*>(side.tl + ((side.cpos + pg) * P + j) * side.H + side.hcol) =
              make_float2(u[pg][2 * h] * s.kq0, u[pg][2 * h + 1] * s.kq1);
      }
    }
  }
}

// The warp's record of a sequence, in the layout of ce_decode.cu's records.
__device__ __forceinline__ void leave(const Params& p, Rows& s, int b, int warp, int lane) {
  const int r = lane >> 2, t = lane & 3;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    s.l0 += __shfl_xor_sync(0xffffffffu, s.l0, o);
    s.l1 += __shfl_xor_sync(0xffffffffu, s.l1, o);
    s.z0 += __shfl_xor_sync(0xffffffffu, s.z0, o);
    s.z1 += __shfl_xor_sync(0xffffffffu, s.z1, o);
  }
  float* rec = p.rec + static_cast<int64_t>(b + blockIdx.x) * REC_FLOATS;
  const int v0 = warp * 8 + 2 * t;
  // accumulators hold sum (p s 2^15 / bound) (c 2^-24), upper nibbles 16-fold;
  // bound 2^9 in two steps that cannot overflow
  const float fb = s.bound * 9.5367431640625e-7f;   // 2^-20
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    rec[v0 * D + q * 16 + r] = fmaf(s.o[q][0] * 536870912.f, fb, s.z0);
    rec[(v0 + 1) * D + q * 16 + r] = fmaf(s.o[q][1] * 536870912.f, fb, s.z1);
    rec[v0 * D + q * 16 + r + 8] = fmaf(s.o[q][2] * 33554432.f, fb, s.z0);
    rec[(v0 + 1) * D + q * 16 + r + 8] = fmaf(s.o[q][3] * 33554432.f, fb, s.z1);
  }
  if (r == 0) {
    rec[REC_ROWS * D + v0] = s.m0;
    rec[REC_ROWS * D + v0 + 1] = s.m1;
    rec[REC_ROWS * D + REC_ROWS + v0] = s.l0;
    rec[REC_ROWS * D + REC_ROWS + v0 + 1] = s.l1;
  }
}

__device__ __forceinline__ int stages_of(const Params& p, int b, int ST) {
  return (decode::seq_tokens(p, b, P) + ST - 1) / ST;
}

// Warps 0..7 consume (warp w: KV head w % G, pages 4 (w / G) .. +3 of each
// stage), warps 8.. produce (stage k by warp 8 + k % NPW).
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM)
    attn_kernel(const Params p, const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NSTAGES * STAGE_BYTES);
  uint64_t* empty = full + NSTAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + NSTAGES);
  int* start_sh = reinterpret_cast<int*>(smem + NSTAGES * STAGE_BYTES + 64);
  int64_t* scan_sh = reinterpret_cast<int64_t*>(smem + NSTAGES * STAGE_BYTES + 128);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G, H = p.H;
  const int ST = WT * (NCW / G);            // tokens per stage
  const int UPS = ST / P;                   // pages per stage
  const int unit_bytes = G * SLICE;

  if (tid == 0) {
    for (int s = 0; s < NSTAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], NCW);
    }
    *abort_flag = 0;
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
  const int64_t excl = decode::block_excl_scan(local, scan_sh, S);
  const int64_t k = blockIdx.x, grid = decode::eff_grid(S, gridDim.x, MIN_STAGES_LOG2);
  const int64_t S_lo = k < grid ? k * S / grid : S, S_hi = k < grid ? (k + 1) * S / grid : S;
  if (blockIdx.x == 0) {
    int64_t run = excl;
    for (int b = lo_b; b < hi_b; ++b) {
      p.prefix[b] = static_cast<int32_t>(run);
      const int n = stages_of(p, b, ST);
      run += n;
      if (n == 0) decode::empty_sequence(p, b);
    }
    if (tid == 0) p.prefix[bs] = static_cast<int32_t>(S);
  }
  if (tid == 0) {
    start_sh[0] = bs;
    start_sh[1] = 0;
  }
  __syncthreads();
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

  int b = start_sh[0], base = start_sh[1];
  int nst = 0, tok_b = 0;
  int64_t ip_b = 0;
  auto load_seq = [&](int bb) {
    tok_b = decode::seq_tokens(p, bb, P);
    nst = (tok_b + ST - 1) / ST;
    ip_b = p.kv_indptr[bb];
  };
  if (b < bs) load_seq(b);

  if (warp >= NCW) {
    // ------------------------------- producers -------------------------------
    // Page indices in 32-entry windows, a third one in flight, as for bf16 pages.
    const int pw = warp - NCW;
    int issued = 0;
    auto fetch = [&](int64_t w0) -> int {
      const int64_t c = w0 + lane;
      return (c >= 0 && c < p.kv_capacity) ? p.kv_indices[c] : -2;
    };
    int64_t w0 = -1;
    int idx_cur = -2, idx_next = -2, idx_ahead = -2;
    for (int64_t x = S_lo; x < S_hi; ++x) {
      while (x >= base + nst) {
        base += nst;
        ++b;
        load_seq(b);
      }
      if (*abort_flag) break;
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
      if (issued % NPW != pw) {
        ++issued;
        continue;
      }
      if (issued >= NSTAGES) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait_or_abort(&empty[s], ((issued / NSTAGES) & 1) ^ 1, p.err, abort_flag);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) {
          *abort_flag = 1;
          break;
        }
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
      if (lane == 0) mbar_arrive_expect_tx(&full[s], __popc(valid) * unit_bytes * 2);
      __syncwarp();
      if (unit >= 0) {
        uint8_t* kd = smem + s * STAGE_BYTES + lane * unit_bytes;
        const int64_t off = static_cast<int64_t>(unit) * unit_bytes;
        bulk_load(kd, k_pool + off, unit_bytes, &full[s]);
        bulk_load(kd + HALF_STAGE, v_pool + off, unit_bytes, &full[s]);
      }
      ++issued;
    }
    // Every load this warp issued lands before the CTA may exit.
    if (lane == 0) {
      for (int it = max(0, issued - NSTAGES); it < issued; ++it)
        if (it % NPW == pw) mbar_wait(&full[it % NSTAGES], (it / NSTAGES) & 1, p.err);
    }
  } else {
    // ------------------------------- consumers -------------------------------
    const int g = warp % G, tb = warp / G;
    const int head = g * GROUP + (lane >> 2);
    Rows st;
    Side side{CE_MODE_NONE, 0, p.kv_capacity, H, g * GROUP + 2 * (lane & 3), p.ul, p.tl};
    int cur_b = -1, s = 0;
    uint32_t ph = 0;
    bool aborted = false;
    for (int64_t x = S_lo; x < S_hi; ++x) {
      while (x >= base + nst) {
        base += nst;
        ++b;
        load_seq(b);
      }
      if (b != cur_b) {
        if (cur_b >= 0) leave(p, st, cur_b, warp, lane);
        cur_b = b;
        clear(st);
        load_query(st, p.q + static_cast<int64_t>(b) * p.q_sb + static_cast<int64_t>(head) * p.q_sh, lane & 3,
                   p.scale_log2);
        side.mode = decode::seq_mode(p, b);
        if (side.mode != CE_MODE_SUM && side.mode != CE_MODE_MAX) side.mode = CE_MODE_NONE;
        if ((side.mode == CE_MODE_SUM && !p.ul) || (side.mode == CE_MODE_MAX && !p.tl)) {
          if (lane == 0 && warp == 0) flag_error(p.err, CE_EW_MODE);
          side.mode = CE_MODE_NONE;
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
      const uint8_t* kb = smem + cs * STAGE_BYTES + tb * PPW * unit_bytes + g * SLICE;
      side.cpos = ip_b + static_cast<int64_t>(j) * UPS + tb * PPW;
      if (mine >= WT)
        tile<false>(st, kb, kb + HALF_STAGE, unit_bytes, WT, lane, side);
      else if (mine > 0)
        tile<true>(st, kb, kb + HALF_STAGE, unit_bytes, mine, lane, side);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[cs]);   // release orders the reads above
    }
    if (cur_b >= 0) leave(p, st, cur_b, warp, lane);
  }
  __syncthreads();
}

}  // namespace kv4
}  // namespace ce

using namespace ce;

namespace {
int check_shape(int32_t bs, int64_t pool_units, int64_t cap, int32_t H, int32_t G, int32_t head_dim, int32_t page_size) {
  if (bs < 0 || pool_units < 0 || cap < 0) return host::fail(CE_ERR_ARG, "ce_kv4_decode: negative size");
  if (head_dim != kv4::D) return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_decode: head_dim must be 64");
  if (G <= 0 || H != kv4::GROUP * G || kv4::NCW % G != 0)
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
  if (!host::set_smem(kv4::attn_kernel, kv4::SMEM_BYTES)) return host::fail(CE_ERR_CUDA, "smem attr");
  kv4::attn_kernel<<<grid, kv4::THREADS, kv4::SMEM_BYTES, st>>>(p, static_cast<const uint8_t*>(k_pool),
                                                                static_cast<const uint8_t*>(v_pool));
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_decode launch");
  return host::launch_combine(p, grid, kv4::P, (score_flags & CE_SCORE_DEFER) != 0, st);
}

int ce::host::kv4_prepare_device() {
  if (!host::set_smem(kv4::attn_kernel, kv4::SMEM_BYTES)) return host::fail_cuda("4-bit decode kernel: set-up");
  return host::kv4_copy_prepare_device();
}
