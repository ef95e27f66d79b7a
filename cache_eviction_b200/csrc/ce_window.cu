// ce_window_prefill: causal attention of extend chunks with a sliding window
// and a few first tokens, over the paged bf16 pools, on the 5th-generation
// tensor cores.
//
//   out_i = softmax over {t <= p, t > p - window or t < first} (and the sink) of
//           scale q_i . k_t,  times v_t,    p = kv_tokens - nq + i
//
// One CTA per (16 queries, KV head, entry): its 128 accumulator rows are the
// 16 queries' 8 heads, which share every key and value tile.  It walks the
// 128-key tiles that hold a visible token of some row (the first tokens'
// tiles, then the window's, which start at a page boundary), in one pass:
//   load warp     K and V tiles in the order the MMA warp takes them, through
//                 a ring of five 16 KB slots (page loads by TMA, or cp.async
//                 gathers for pages under 8 tokens)
//   MMA warp      S(t) = Q K^T into tensor memory, then O += P(t-1) V
//   softmax warps one thread per row: S from tensor memory, running maximum
//                 and sum, P = 2^(s - m) in bf16 back into tensor memory as the
//                 A operand of the second product.  O is rescaled only when a
//                 row's maximum has grown by more than 2^8 since the last
//                 rescale (P stays below 2^8, its relative precision and the
//                 fp32 sum's are the same), so S(t+1) and P V(t) run under
//                 the exponentials of tile t.
// Two CTAs share an SM (256 TMEM columns and 97 KB each), so that one's
// exponentials cover the other's waits.  The exponentials bound the kernel:
// one per (row, key) of a tile against 2 x 128 x 64 multiply-adds, so a share of
// them runs as a polynomial on the FMA pipes.  P in bf16 is rounded by at most
// 2^-9 of itself, less than the output's own rounding makes of it on average;
// maxima, sums and O are fp32.
//
// What a row must not see must not reach it: a masked key's logit is replaced
// before the maximum, and a masked value meets P = 0, which is no help if it
// is infinite or NaN.  So in a tile that some row sees only in part the MMA
// warp clears the values that no row sees (a page's unwritten slots, pages that
// were not loaded) and any value that is not finite, noting its token; a row
// that does see such a token gets NaN at the end.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "ce_common.cuh"
#include "ce_host.h"

namespace ce {
namespace window {

constexpr int D = 64;
constexpr int GROUP = 8;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int BM = 128;                  // accumulator rows
constexpr int BN = 128;                  // keys per tile
constexpr int QT = BM / GROUP;           // 16 queries per CTA
constexpr int TILE = 128 * 128;          // 128 rows x 128 B
constexpr int SLOTS = 5;                 // ring of K and V tiles
constexpr int LAG = 3;                   // cp.async tiles in flight before one is published
constexpr int SM_WARPS = 4;              // softmax: TMEM lanes 32 w .. +31
constexpr int LOAD_WARP = SM_WARPS, MMA_WARP = SM_WARPS + 1;
constexpr int THREADS = 32 * (SM_WARPS + 2);
constexpr uint32_t TMEM_COLS = 256, P_COL = 128, O_COL = 192;
constexpr uint32_t IDESC_S = f16_idesc(BM, BN);
constexpr uint32_t IDESC_PV = f16_idesc(BM, D) | kIdescBMajorMN;
constexpr float LAZY = 8.f;              // log2 growth of a maximum that is let through
constexpr int MAX_EDGE = 12;             // tiles of a CTA that some row may see in part

struct Params {
  const __nv_bfloat16 *k, *v;
  int64_t pool_units;
  const int32_t *qo_indptr, *kv_indptr, *kv_indices, *kv_tokens;
  int64_t kv_capacity;
  const float* sinks;
  float scale2;           // sm_scale * log2(e)
  int G, P;
  int total_q, max_q, max_tokens;
  int window, first;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  int32_t* err;
};

struct Sync {
  uint64_t full[SLOTS], empty[SLOTS];
  uint64_t sfull, sempty, pfull, pempty;
  uint64_t once, odone, mma_done;
  uint32_t tmem;
  int abort;
  int edges;                      // tiles whose values the MMA warp looked through
  int edge_key[MAX_EDGE];         // their first token
  uint32_t edge_bad[MAX_EDGE][4]; // their tokens with a value that is not finite
};

// The keys a CTA's rows (positions p_lo .. p_hi) see, as 128-key tiles.
struct Span {
  int p_lo, p_hi, lo, first, window;   // lo: first key in some row's window
  int head, start, ntiles;             // tiles 0 .. head-1 at 128 t, the rest from `start` on
  __device__ __forceinline__ Span(const Params& p, int plo, int phi) : p_lo(plo), p_hi(phi), window(p.window) {
    const int kend = p_hi + 1;
    lo = window < 0 ? 0 : max(0, p_lo - window + 1);
    first = window < 0 ? 0 : min(p.first, kend);
    head = (first + BN - 1) / BN;
    const int align = max(16, p.P);
    start = lo / align * align;
    if (start <= head * BN) {   // the window reaches the first tokens' tiles
      start = first > 0 ? 0 : start;
      head = 0;
    }
    ntiles = head + (kend - start + BN - 1) / BN;
  }
  __device__ __forceinline__ int key(int t) const { return t < head ? t * BN : start + (t - head) * BN; }
  // Whether some row sees a key of [k, k + n) / key k.
  __device__ __forceinline__ bool some(int k, int n) const { return k <= p_hi && (k + n > lo || k < first); }
  // Whether every row sees every key of the tile at k.
  __device__ __forceinline__ bool whole(int k) const {
    return k + BN - 1 <= p_lo && (window < 0 || k > p_hi - window || k + BN <= first);
  }
  __device__ __forceinline__ bool sees(int pos, int k) const {
    return k <= pos && (window < 0 || k > pos - window || k < first);
  }
};

__device__ __forceinline__ bool entry_ok(const Params& p, int b, int& qbeg, int& nq, int& ntok, int& list0) {
  qbeg = p.qo_indptr[b];
  nq = p.qo_indptr[b + 1] - qbeg;
  ntok = p.kv_tokens[b];
  list0 = p.kv_indptr[b];
  const int64_t units = (static_cast<int64_t>(ntok) + p.P - 1) / p.P;
  const bool ok = qbeg >= 0 && nq >= 0 && qbeg + static_cast<int64_t>(nq) <= p.total_q && nq <= p.max_q &&
                  ntok <= p.max_tokens && ntok >= nq && list0 >= 0 && list0 + units <= p.kv_capacity &&
                  units <= p.kv_indptr[b + 1] - list0;
  if (!ok && threadIdx.x == 0 && blockIdx.x == 0) flag_error(p.err, CE_EW_SHAPE);
  return ok;
}

// Unit of the list's token t, or -1 (outside the pool: flagged).
__device__ __forceinline__ int token_unit(const Params& p, int list0, int t) {
  const int unit = p.kv_indices[list0 + t / p.P];
  if (unit >= 0 && unit < p.pool_units) return unit;
  flag_error(p.err, CE_EW_INDEX);
  return -1;
}

// Keys k0 .. k0 + 127 of head g by page loads (pages of at least 8 rows, each
// on a 1024-byte boundary of the tile), completing on `bar`.
__device__ __forceinline__ void tma_tile(const Params& p, const Span& sp, const CUtensorMap* map, uint8_t* tile,
                                         uint64_t* bar, int list0, int k0, int g, int lane) {
  const int t = k0 + lane * p.P;
  const int unit = lane < BN / p.P && sp.some(t, p.P) ? token_unit(p, list0, t) : -1;
  const unsigned valid = __ballot_sync(0xffffffffu, unit >= 0);
  if (lane == 0) mbar_arrive_expect_tx(bar, __popc(valid) * p.P * 128);
  __syncwarp();
  if (unit >= 0) tma_load_2d(tile + lane * p.P * 128, map, 0, (unit * p.G + g) * p.P, bar);
}

// The same for smaller pages by cp.async; rows that no query sees are zeros.
__device__ __forceinline__ void copy_tile(const Params& p, const Span& sp, const __nv_bfloat16* pool, uint32_t tile,
                                          int list0, int k0, int g, int lane) {
  int u[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int t = k0 + lane + 32 * k;
    u[k] = sp.some(t, 1) ? token_unit(p, list0, t) : -1;
  }
  const int c = lane & 7;
#pragma unroll
  for (int j = 0; j < BN / 4; ++j) {
    const int r = (lane >> 3) + 4 * j;
    const int unit = __shfl_sync(0xffffffffu, u[j >> 3], r & 31);
    const bool ok = unit >= 0;
    const __nv_bfloat16* src =
        ok ? pool + ((static_cast<int64_t>(unit) * p.G + g) * p.P + (k0 + r) % p.P) * D + c * 8 : pool;
    cp_async16(tile + swz(r, c), src, ok);
  }
}

// Halves of a bf16 pair that are not finite, as masks.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

// A partly visible value tile (keys from k on) made safe for P = 0 (one warp).
__device__ __forceinline__ void clean_values(const Span& sp, uint8_t* tile, int k, Sync* sy, int lane) {
  const int e = sy->edges;
  __syncwarp();
  uint32_t bad[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = w * 32 + i * 4 + (lane >> 3);
      uint4* at = reinterpret_cast<uint4*>(tile + row * 128 + (lane & 7) * 16);
      if (!sp.some(k + row, 1)) {
        *at = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      uint4 x = *at;
      const uint32_t top = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                    __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
      if ((top & 0xffffu) >= 0x7f80u || (top >> 16) >= 0x7f80u) {
        x.x &= ~not_finite(x.x);
        x.y &= ~not_finite(x.y);
        x.z &= ~not_finite(x.z);
        x.w &= ~not_finite(x.w);
        *at = x;
        bad[w] |= 1u << (row & 31);
      }
    }
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) bad[w] = __reduce_or_sync(0xffffffffu, bad[w]);
  if (lane == 0 && e < MAX_EDGE) {
    sy->edge_key[e] = k;
#pragma unroll
    for (int w = 0; w < 4; ++w) sy->edge_bad[e][w] = bad[w];
    if (bad[0] | bad[1] | bad[2] | bad[3]) sy->edges = e + 1;   // a clean tile's entry is used again
  }
  fence_proxy_async();
  __syncwarp();
}

__device__ __forceinline__ void tmem_st16_async(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// P = 2^(scale2 v - mu) of a row's tile in bf16 into tensor memory; returns its
// sum.  A quarter of the exponentials run as a polynomial, which never gives
// an exact 0, so a tile with masked keys (-inf) takes none.
template <bool EDGE>
__device__ __forceinline__ float weights(const float (&v)[BN], float scale2, float mu, uint32_t col) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < BN; c += 32) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float x = fast_exp2(fmaf(v[c + i], scale2, -mu));
      const float a = fmaf(v[c + i + 1], scale2, -mu);
      const float y = !EDGE && (i & 2) ? poly_exp2(a) : fast_exp2(a);
      sum[i & 2] += x;
      sum[(i & 2) + 1] += y;
      const __nv_bfloat162 xy = __floats2bfloat162_rn(x, y);
      w[i / 2] = *reinterpret_cast<const uint32_t*>(&xy);
    }
    tmem_st16_async(col + c / 2, w);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

constexpr int SMEM = 1024 + TILE + SLOTS * TILE + static_cast<int>(sizeof(Sync));
// At most two CTAs fit on an SM (2 x 256 TMEM columns = all 512): tcgen05.alloc never waits.
static_assert(2 * (SMEM + 1024) <= 228 * 1024 && 3 * (SMEM + 1024) > 228 * 1024, "two CTAs per SM");

__global__ void __launch_bounds__(THREADS, 2)
    attend_kernel(const Params p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  const int b = blockIdx.z, g = blockIdx.y;
  int qbeg, nq, ntok, list0;
  if (!entry_ok(p, b, qbeg, nq, ntok, list0)) return;
  // the longest rows first: the last queries see the most keys
  const int q0 = (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)) * QT;
  if (q0 >= nq) return;
  const int prefix = ntok - nq;
  const Span sp(p, prefix + q0, prefix + min(nq, q0 + QT) - 1);
  const int ntiles = sp.ntiles;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  const uint32_t qtile = smem_addr(sm);
  const uint32_t ring = qtile + TILE;
  Sync* sy = reinterpret_cast<Sync*>(sm + TILE + SLOTS * TILE);
  volatile int* abort = &sy->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sy->full[s], 1);
      mbar_init(&sy->empty[s], 1);
    }
    mbar_init(&sy->sfull, 1);
    mbar_init(&sy->sempty, SM_WARPS);
    mbar_init(&sy->pfull, SM_WARPS);
    mbar_init(&sy->pempty, 1);
    mbar_init(&sy->once, 1);
    mbar_init(&sy->odone, 2);   // the last product and the MMA thread (its notes are in place)
    mbar_init(&sy->mma_done, 1);
    sy->abort = 0;
    sy->edges = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) tmem_alloc(&sy->tmem, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sy->tmem;

  // Ring order: K(0), then for t = 1 ..: K(t), V(t - 1); V(ntiles - 1) last.
  // Position i of it is K(0) for i = 0, K((i + 1) / 2) for odd i < 2 ntiles - 1
  // and V(i / 2 - 1) for even i > 0; the last one, 2 ntiles - 1, is V(ntiles - 1).
  if (warp == LOAD_WARP) {
    const int total = 2 * ntiles;
    const bool tma = p.P >= 8;
    if (lane == 0) {
      mbar_arrive_expect_tx(&sy->once, TILE);
      tma_load_3d(sm, &qmap, 0, g * GROUP, qbeg + q0, &sy->once);
    }
    int i = 0;
    for (; i < total; ++i) {
      const int s = i % SLOTS;
      const bool is_v = i > 0 && ((i & 1) == 0 || i == total - 1);
      const int t = i == 0 ? 0 : i == total - 1 ? ntiles - 1 : is_v ? i / 2 - 1 : (i + 1) / 2;
      if (i >= SLOTS && !warp_wait(&sy->empty[s], ((i / SLOTS) & 1) ^ 1, p.err, abort, lane)) {
        *abort = 1;
        break;
      }
      if (tma) {
        tma_tile(p, sp, is_v ? &vmap : &kmap, sm + TILE + s * TILE, &sy->full[s], list0, sp.key(t), g, lane);
        continue;
      }
      copy_tile(p, sp, is_v ? p.v : p.k, ring + s * TILE, list0, sp.key(t), g, lane);
      cp_async_commit();
      if (i >= LAG) {
        cp_async_wait<LAG>();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sy->full[(i - LAG) % SLOTS]);
      }
    }
    if (!tma) {
      cp_async_wait<0>();
      fence_proxy_async();
      __syncwarp();
      if (lane == 0 && !*abort)
        for (int u = max(0, i - LAG); u < i; ++u) mbar_arrive(&sy->full[u % SLOTS]);
    }
    if (lane == 0) {   // every issued load lands before the CTA may exit
      if (tma)
        for (int u = max(0, i - SLOTS); u < i; ++u) mbar_wait(&sy->full[u % SLOTS], (u / SLOTS) & 1, p.err);
      mbar_wait(&sy->once, 0, p.err);
    }
  } else if (warp == MMA_WARP) {
    bool issued = false, ok = warp_wait(&sy->once, 0, p.err, abort, lane);
    int i = 0;   // ring position
    for (int t = 0; t <= ntiles && ok; ++t) {
      if (t < ntiles) {
        const int s = i % SLOTS;
        ok = warp_wait(&sy->full[s], (i / SLOTS) & 1, p.err, abort, lane) &&
             (t == 0 || warp_wait(&sy->sempty, (t - 1) & 1, p.err, abort, lane));
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint64_t qdesc = sw128_desc(qtile), kdesc = sw128_desc(ring + s * TILE);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) tc_mma(tmem, qdesc + 2 * kk, kdesc + 2 * kk, IDESC_S, kk > 0);
          tc_commit(&sy->sfull);
          tc_commit(&sy->empty[s]);
        }
        issued = true;
        ++i;
      }
      if (t >= 1) {
        const int u = t - 1, s = i % SLOTS;
        ok = warp_wait(&sy->full[s], (i / SLOTS) & 1, p.err, abort, lane);
        if (!ok) break;
        if (!sp.whole(sp.key(u))) clean_values(sp, sm + TILE + s * TILE, sp.key(u), sy, lane);
        ok = warp_wait(&sy->pfull, u & 1, p.err, abort, lane);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t vt = ring + s * TILE;
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            tc_mma_ts(tmem + O_COL, tmem + P_COL + kk * 8, sw128_mn_desc(vt + kk * 2048), IDESC_PV, u > 0 || kk > 0);
          tc_commit(&sy->pempty);
          tc_commit(&sy->empty[s]);
        }
        ++i;
      }
    }
    if (lane == 0) {
      if (ok) {
        mbar_arrive(&sy->odone);
        tc_commit(&sy->odone);
      } else {
        *abort = 1;
      }
      if (issued) {   // every MMA completes before the tensor memory may be freed
        tc_commit(&sy->mma_done);
        mbar_wait(&sy->mma_done, 0, p.err);
      }
    }
    __syncwarp();
  } else {
    const int r = warp * 32 + lane;              // accumulator row = TMEM lane
    const int q = q0 + r / GROUP;
    const int h = g * GROUP + r % GROUP;
    const int pos = prefix + min(q, nq - 1);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int t = 0; t < ntiles; ++t) {
      if (!warp_wait(&sy->sfull, t & 1, p.err, abort, lane)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float v[BN];
      __syncwarp();
#pragma unroll
      for (int c = 0; c < BN; c += 32) tmem_ld32_async(lanes + c, v + c);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sy->sempty);   // the values are in registers
      const int k0 = sp.key(t);
      const bool edge = !sp.whole(k0);
      if (edge) {
        const int hi = pos - k0, lo = sp.window < 0 || hi < 0 ? -1 : hi - sp.window, fi = sp.first - k0;
#pragma unroll
        for (int i = 0; i < BN; ++i) v[i] = (i <= hi && (i > lo || i < fi)) ? v[i] : -INFINITY;
      }
      float mx[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mx[i] = v[i];
#pragma unroll
      for (int i = 8; i < BN; ++i) mx[i & 7] = fmaxf(mx[i & 7], v[i]);
      const float mt = p.scale2 * fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                        fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
      if (t >= 1 && !warp_wait(&sy->pempty, (t - 1) & 1, p.err, abort, lane)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool grow = mt > m + LAZY || (m == -INFINITY && mt > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float mn = grow ? mt : m;
        const float a = m == -INFINITY ? 0.f : fast_exp2(m - mn);
        l *= a;
        m = mn;
        if (t >= 1) {   // P V(t - 1) has completed: O is at rest
          float o[32];
          __syncwarp();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            tmem_ld32(lanes + O_COL + c, o);
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(o[i] * a);
            tmem_st16_async(lanes + O_COL + c, w);
            tmem_st16_async(lanes + O_COL + c + 16, w + 16);
          }
        }
      }
      const float mu = m == -INFINITY ? 0.f : m;
      __syncwarp();
      l += edge ? weights<true>(v, p.scale2, mu, lanes + P_COL) : weights<false>(v, p.scale2, mu, lanes + P_COL);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sy->pfull);
    }
    if (!ok) *abort = 1;
    if (ok && warp_wait(&sy->odone, 0, p.err, abort, lane)) {
      tc_fence_after();
      float o[D];
      __syncwarp();
      tmem_ld32_async(lanes + O_COL, o);
      tmem_ld32_async(lanes + O_COL + 32, o + 32);
      tmem_ld_wait();
      if (p.sinks) l += exp2f(p.sinks[h] * LOG2E - m);
      float f = 1.f / l;
      for (int e = 0; e < min(sy->edges, MAX_EDGE); ++e)
        for (int w = 0; w < 4; ++w)
          for (uint32_t bad = sy->edge_bad[e][w]; bad; bad &= bad - 1)
            if (sp.sees(pos, sy->edge_key[e] + w * 32 + __ffs(bad) - 1)) f = __int_as_float(0x7fc00000);
      if (q < nq) {
        uint4* dst = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(qbeg + q) * p.o_st +
                                              static_cast<int64_t>(h) * p.o_sh);
#pragma unroll
        for (int c = 0; c < D; c += 8) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(o[c + 2 * i] * f, o[c + 2 * i + 1] * f);
            w[i] = *reinterpret_cast<const uint32_t*>(&x);
          }
          dst[c / 8] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace window
}  // namespace ce

using namespace ce;

extern "C" int ce_window_prefill(const void* q, int64_t q_st, int64_t q_sh, const void* k_pool, const void* v_pool,
                                 int64_t pool_units, const int32_t* qo_indptr, const int32_t* kv_indptr,
                                 const int32_t* kv_indices, const int32_t* kv_tokens, int64_t kv_capacity,
                                 const float* sinks, float sm_scale, int32_t bs, int32_t num_q_heads,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int32_t total_q,
                                 int32_t max_q, int32_t max_tokens, int32_t window, int32_t first, void* out,
                                 int64_t o_st, int64_t o_sh, int32_t* err, void* stream) {
  using namespace ce::window;
  if (bs < 0 || total_q < 0 || max_q < 0 || max_tokens < 0 || pool_units < 0 || kv_capacity < 0)
    return host::fail(CE_ERR_ARG, "ce_window_prefill: negative size");
  if (window == 0 || window < -1 || first < 0)
    return host::fail(CE_ERR_ARG, "ce_window_prefill: window must be at least 1 (or -1: none), first at least 0");
  if (!(sm_scale > 0.f)) return host::fail(CE_ERR_ARG, "ce_window_prefill: sm_scale must be positive");
  if (head_dim != D || num_kv_heads <= 0 || num_q_heads != GROUP * num_kv_heads)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_window_prefill: needs head_dim 64 and 8 query heads per KV head");
  if (page_size <= 0 || page_size > 64 || 64 % page_size != 0)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_window_prefill: page_size must divide 64");
  if (q_sh % 8 != 0 || q_st % 8 != 0 || q_sh < D || q_st < static_cast<int64_t>(num_q_heads) * q_sh || o_sh % 8 != 0 ||
      o_st % 8 != 0)
    return host::fail(CE_ERR_ARG, "ce_window_prefill: strides must be multiples of 8 elements, heads inside a token's row");
  if (bs == 0 || max_q == 0 || total_q == 0) return CE_OK;
  if (!q || !k_pool || !v_pool || !qo_indptr || !kv_indptr || !kv_indices || !kv_tokens || !out)
    return host::fail(CE_ERR_ARG, "ce_window_prefill: null pointer");
  if (pool_units == 0) return host::fail(CE_ERR_ARG, "ce_window_prefill: empty pool");
  if (bs > 65535 || num_kv_heads > 65535)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_window_prefill: more than 65535 entries or heads");
  if (pool_units * num_kv_heads * page_size > INT32_MAX)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_window_prefill: pool rows exceed 2^31");
  if (max_tokens > INT32_MAX - 2 * BN)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_window_prefill: too many tokens");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return host::fail(CE_ERR_ARG, "ce_window_prefill: q, pools and out need 16-byte alignment");
  CUtensorMap qmap, kmap, vmap;
  {
    // Q as [total_q][H][64] with byte strides; box = 16 queries x 8 heads x 64.
    const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(num_q_heads),
                              static_cast<uint64_t>(total_q)};
    const uint64_t strides[2] = {static_cast<uint64_t>(q_sh) * 2, static_cast<uint64_t>(q_st) * 2};
    const uint32_t box[3] = {static_cast<uint32_t>(D), GROUP, QT};
    if (!host::encode_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, dims, strides, box, true))
      return host::fail(CE_ERR_CUDA, "ce_window_prefill: query tensor map");
  }
  // Pools as [units * G * page, 64] rows; box = one page of one head.
  const uint64_t rows = static_cast<uint64_t>(pool_units) * num_kv_heads * page_size;
  if (!host::encode_rows_map(&kmap, k_pool, rows, D, static_cast<uint32_t>(page_size)) ||
      !host::encode_rows_map(&vmap, v_pool, rows, D, static_cast<uint32_t>(page_size)))
    return host::fail(CE_ERR_CUDA, "ce_window_prefill: pool tensor maps");
  Params p{};
  p.k = static_cast<const __nv_bfloat16*>(k_pool);
  p.v = static_cast<const __nv_bfloat16*>(v_pool);
  p.pool_units = pool_units;
  p.qo_indptr = qo_indptr;
  p.kv_indptr = kv_indptr;
  p.kv_indices = kv_indices;
  p.kv_tokens = kv_tokens;
  p.kv_capacity = kv_capacity;
  p.sinks = sinks;
  p.scale2 = sm_scale * LOG2E;
  p.G = num_kv_heads;
  p.P = page_size;
  p.total_q = total_q;
  p.max_q = max_q;
  p.max_tokens = max_tokens;
  p.window = window;
  p.first = first;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.err = err;
  if (!host::set_smem(attend_kernel, SMEM)) return host::fail(CE_ERR_CUDA, "ce_window_prefill: smem attr");
  const dim3 grid((max_q + QT - 1) / QT, num_kv_heads, bs);
  attend_kernel<<<grid, THREADS, SMEM, static_cast<cudaStream_t>(stream)>>>(p, qmap, kmap, vmap);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_window_prefill launch");
  return CE_OK;
}
