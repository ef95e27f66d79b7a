// ce_window_prefill: causal attention of extend chunks with a sliding window
// and a few first tokens, over the paged bf16 pools, on the 5th-generation
// tensor cores.
//
//   out_i = softmax over {t <= p, t > p - window or t < first} (and the sink) of
//           scale q_i . k_t,  times v_t,    p = kv_tokens - nq + i
//
// One CTA per (32 queries, KV head, entry), two tiles of 16 queries whose 8
// heads are a tile's 128 accumulator rows and share every key and value tile.
// It walks the 128-key tiles that hold a visible token of some row (the first
// tokens' tiles, then the window's, which start at a page boundary), in one pass:
//   load warps    K tiles through one ring of 16 KB slots, V tiles through
//                 another (page loads by TMA, or cp.async gathers for pages
//                 under 8 tokens), page indices read a tile ahead
//   S warp        S(t) = Q K^T of both query tiles into tensor memory, each as
//                 soon as its S(t-1) is read
//   PV warp       O += P(t) V(t) of each once its weights are in place
//   softmax warps eight per query tile, two threads per row, 64 keys each: S from
//                 tensor memory, running maximum (exchanged through shared
//                 memory) and sum, P = 2^(s - m) in bf16 back into tensor
//                 memory as the A operand of the second product.  O is
//                 rescaled only when a row's maximum has grown by more than
//                 2^8 since the last rescale (P stays below 2^8, its relative
//                 precision and the fp32 sum's are the same).
// The exponentials bound the kernel (one per row and key on a unit of 16 per
// clock and SM: 1,024 clocks per tile, against 768 of the tensor cores), so the
// two query tiles take turns at them: while one computes its weights the
// other's waits, reads and maxima go on.  Left to themselves (two CTAs per SM)
// the tiles fell into step, both at the exponentials and then both waiting.
// (Taking a share of the exponentials as a polynomial on the FMA pipes was
// slower at every share.)  P in bf16 is rounded by at most 2^-9 of itself, less
// than the output's own rounding makes of it on average; maxima, sums and O
// are fp32.
//
// What a row must not see must not reach it: a masked key's logit is replaced
// before the maximum, and a masked value meets P = 0, which is no help if it
// is infinite or NaN.  So in a tile that some row sees only in part the PV
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
constexpr int QT = BM / GROUP;           // 16 queries per tile
constexpr int TILES = 2;                 // query tiles per CTA
constexpr int TILE = 128 * 128;          // 128 rows x 128 B
constexpr int KS = 5, VS = 5;            // ring slots of K and V tiles
constexpr int LAG = 3;                   // cp.async tiles in flight before one is published
constexpr int SM_WARPS = 8;              // softmax, per query tile: TMEM lanes 32 (w % 4) .. +31, keys 64 (w / 4) .. +63
constexpr int HALF = BN / 2;             // keys of a softmax thread
constexpr int K_WARP = TILES * SM_WARPS, V_WARP = K_WARP + 1, S_WARP = K_WARP + 2;   // and the PV warp
constexpr int THREADS = 32 * (TILES * SM_WARPS + 4);
constexpr uint32_t TMEM_TILE = 256, TMEM_COLS = TILES * TMEM_TILE, P_COL = 128, O_COL = 192;   // S | P | O of each tile
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
  uint64_t kfull[KS], kempty[KS], vfull[VS], vempty[VS];
  uint64_t sfull[TILES], sempty[TILES], pfull[TILES], pempty[TILES];
  uint64_t once, odone, s_done, pv_done;
  uint32_t tmem;
  int abort;
  float top[TILES][2][2][BM];     // by query tile, key tile parity and half: the rows' maxima; at the end their sums
  int edges;                      // tiles in whose values the PV warp found some that are not finite
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

// A load warp's tiles of one pool through its ring.  PAGE: tokens per page, or
// 0 for any size that divides 64.
template <int PAGE, int SLOTS>
__device__ __forceinline__ void load_tiles(const Params& p, const Span& sp, const CUtensorMap* map,
                                           const __nv_bfloat16* pool, uint8_t* ring, uint64_t* full, uint64_t* empty,
                                           int list0, int g, int lane, volatile int* abort) {
  const int P = PAGE ? PAGE : p.P;
  const bool tma = P >= 8;
  // Pages of at least 8 rows: lane i < 128 / P the tile's page i.  Smaller ones:
  // lane i keys i, i + 32, i + 64 and i + 96.
  auto unit_of = [&](int k) -> int {   // unit holding key k, -1 if no row sees it
    return sp.some(k, tma ? P : 1) ? p.kv_indices[list0 + k / P] : -1;
  };
  auto checked = [&](int unit, int k) -> int {
    if (unit >= 0 && unit < p.pool_units) return unit;
    if (sp.some(k, tma ? P : 1)) flag_error(p.err, CE_EW_INDEX);
    return -1;
  };
  int t = 0;
  if (tma) {
    const int pages = BN / P;
    int next = lane < pages ? unit_of(sp.key(0) + lane * P) : -1;
    for (; t < sp.ntiles; ++t) {
      const int s = t % SLOTS, k0 = sp.key(t) + lane * P;
      const int unit = lane < pages ? checked(next, k0) : -1;
      if (t + 1 < sp.ntiles) next = lane < pages ? unit_of(sp.key(t + 1) + lane * P) : -1;
      const unsigned valid = __ballot_sync(0xffffffffu, unit >= 0);
      if (t >= SLOTS && !warp_wait_quiet(&empty[s], ((t / SLOTS) & 1) ^ 1, p.err, abort, lane)) {
        *abort = 1;
        break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&full[s], __popc(valid) * P * 128);
      __syncwarp();
      if (unit >= 0) tma_load_2d(ring + s * TILE + lane * P * 128, map, 0, (unit * p.G + g) * P, &full[s]);
    }
    if (lane == 0)   // every issued load lands before the CTA may exit
      for (int u = max(0, t - SLOTS); u < t; ++u) mbar_wait(&full[u % SLOTS], (u / SLOTS) & 1, p.err);
    return;
  }
  if constexpr (PAGE == 0) {
    for (; t < sp.ntiles; ++t) {
      const int s = t % SLOTS, k0 = sp.key(t);
      int u[4];
  #pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = unit_of(k0 + lane + 32 * i);
  #pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = checked(u[i], k0 + lane + 32 * i);
      if (t >= SLOTS && !warp_wait_quiet(&empty[s], ((t / SLOTS) & 1) ^ 1, p.err, abort, lane)) {
        *abort = 1;
        break;
      }
      const int c = lane & 7;
  #pragma unroll 4
      for (int j = 0; j < BN / 4; ++j) {
        const int r = (lane >> 3) + 4 * j;
        const int from = (j >> 3) == 0 ? u[0] : (j >> 3) == 1 ? u[1] : (j >> 3) == 2 ? u[2] : u[3];
        const int unit = __shfl_sync(0xffffffffu, from, r & 31);
        const bool ok = unit >= 0;   // rows that no query sees are zeros
        const __nv_bfloat16* src =
            ok ? pool + ((static_cast<int64_t>(unit) * p.G + g) * P + (k0 + r) % P) * D + c * 8 : pool;
        cp_async16(smem_addr(ring) + s * TILE + swz(r, c), src, ok);
      }
      cp_async_commit();
      if (t >= LAG) {
        cp_async_wait<LAG>();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[(t - LAG) % SLOTS]);
      }
    }
    cp_async_wait<0>();
    fence_proxy_async();
    __syncwarp();
    if (lane == 0 && !*abort)
      for (int u = max(0, t - LAG); u < t; ++u) mbar_arrive(&full[u % SLOTS]);
  }
}

// Halves of a bf16 pair that are not finite, as masks.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

// 0 * w added to acc, per half: NaN from the first value that is not finite on.
__device__ __forceinline__ uint32_t taint(uint32_t w, uint32_t acc) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(acc));
  return d;
}

// A partly visible value tile (keys from k on) made safe for P = 0, by one warp:
// rows that no query sees are cleared, then values that are not finite, whose
// tokens are noted.
__device__ __forceinline__ void clean_values(const Span& sp, uint8_t* tile, int k, Sync* sy, int lane) {
  const int e = sy->edges;
  __syncwarp();
  uint8_t* mine = tile + (lane >> 3) * 128 + (lane & 7) * 16;
  const int row0 = lane >> 3, end = sp.p_hi + 1 - k, from = sp.lo - k, head = sp.first - k;
  uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i0 = 0; i0 < BN / 4; i0 += 8) {
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(mine + (i0 + i) * 512);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = (i0 + i) * 4 + row0;
      if (row >= end || (row < from && row >= head)) {   // no query sees it
        *reinterpret_cast<uint4*>(mine + (i0 + i) * 512) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        acc[0] = taint(x[i].x, acc[0]);
        acc[1] = taint(x[i].y, acc[1]);
        acc[2] = taint(x[i].z, acc[2]);
        acc[3] = taint(x[i].w, acc[3]);
      }
    }
  }
  __syncwarp();
  const uint32_t found = not_finite(acc[0]) | not_finite(acc[1]) | not_finite(acc[2]) | not_finite(acc[3]);
  if (__any_sync(0xffffffffu, found != 0u)) {
    uint32_t bad[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const int row = w * 32 + i * 4;
        uint4* at = reinterpret_cast<uint4*>(mine + row * 128);
        uint4 x = *at;
        const uint4 nf = make_uint4(not_finite(x.x), not_finite(x.y), not_finite(x.z), not_finite(x.w));
        if (nf.x | nf.y | nf.z | nf.w) {
          *at = make_uint4(x.x & ~nf.x, x.y & ~nf.y, x.z & ~nf.z, x.w & ~nf.w);
          bad[w] |= 1u << (i * 4 + (lane >> 3));
        }
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) bad[w] = __reduce_or_sync(0xffffffffu, bad[w]);
    if (lane == 0 && e < MAX_EDGE) {
      sy->edge_key[e] = k;
#pragma unroll
      for (int w = 0; w < 4; ++w) sy->edge_bad[e][w] = bad[w];
      sy->edges = e + 1;
    }
  }
  fence_proxy_async();
  __syncwarp();
}

// 8 consecutive fp32 columns of this thread's TMEM lane, waited for.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
  tmem_ld_wait();
}

// P = 2^(scale2 v - mu) of 32 of a row's keys in bf16 into tensor memory;
// returns their sum.
__device__ __forceinline__ float weights(const float (&v)[32], float scale2, float mu, uint32_t col) {
  const uint64_t sc = pair(scale2, scale2), base = pair(-mu, -mu);
  uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < 32; c += 16) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float e0, e1;
      split(fma2(pair(v[c + 2 * i], v[c + 2 * i + 1]), sc, base), e0, e1);
      e0 = fast_exp2(e0);
      e1 = fast_exp2(e1);
      sum[i & 1] = add2(sum[i & 1], pair(e0, e1));
      const __nv_bfloat162 xy = __floats2bfloat162_rn(e0, e1);
      w[i] = *reinterpret_cast<const uint32_t*>(&xy);
    }
    tmem_st8_async(col + c / 2, w);
  }
  float a, b;
  split(add2(sum[0], sum[1]), a, b);
  return a + b;
}

// The two warps of a query tile's row quarter (named barriers 1 to 8).
__device__ __forceinline__ void quarter_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id + 1) : "memory"); }
// Turns at the exponentials (named barriers 9 and 10): query tile x waits for
// its turn, and gives the other its.
__device__ __forceinline__ void turn_wait(int x) {
  asm volatile("bar.sync %0, %1;" ::"r"(9 + x), "n"(2 * SM_WARPS * 32) : "memory");
}
__device__ __forceinline__ void turn_give(int x) {
  asm volatile("bar.arrive %0, %1;" ::"r"(9 + x), "n"(2 * SM_WARPS * 32) : "memory");
}

constexpr int SMEM = 1024 + (TILES + KS + VS) * TILE + static_cast<int>(sizeof(Sync));
// One CTA per SM (it holds all 512 TMEM columns): tcgen05.alloc never waits.
static_assert(SMEM <= 227 * 1024 && 2 * SMEM > 228 * 1024, "one CTA per SM");

template <int PAGE>
__global__ void __launch_bounds__(THREADS, 1)
    attend_kernel(const Params p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  const int b = blockIdx.z, g = blockIdx.y;
  int qbeg, nq, ntok, list0;
  if (!entry_ok(p, b, qbeg, nq, ntok, list0)) return;
  // the longest rows first: the last queries see the most keys
  const int q0 = (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)) * (TILES * QT);
  if (q0 >= nq) return;
  const int prefix = ntok - nq;
  const int groups = nq - q0 > QT ? 2 : 1;   // query tiles with a query
  const Span sp(p, prefix + q0, prefix + min(nq, q0 + TILES * QT) - 1);
  const int ntiles = sp.ntiles;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  const uint32_t qtile = smem_addr(sm);
  uint8_t *kring = sm + TILES * TILE, *vring = kring + KS * TILE;
  Sync* sy = reinterpret_cast<Sync*>(vring + VS * TILE);
  volatile int* abort = &sy->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < KS; ++i) {
      mbar_init(&sy->kfull[i], 1);
      mbar_init(&sy->kempty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&sy->vfull[i], 1);
      mbar_init(&sy->vempty[i], 1);
    }
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&sy->sfull[i], 1);
      mbar_init(&sy->sempty[i], SM_WARPS);
      mbar_init(&sy->pfull[i], SM_WARPS);
      mbar_init(&sy->pempty[i], 1);
    }
    mbar_init(&sy->once, 1);
    mbar_init(&sy->odone, 2);   // the last product and the PV thread (its notes are in place)
    mbar_init(&sy->s_done, 1);
    mbar_init(&sy->pv_done, 1);
    sy->abort = 0;
    sy->edges = 0;
    fence_mbar_init();
  }
  if (warp == S_WARP) tmem_alloc(&sy->tmem, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sy->tmem;

  if (warp >= K_WARP) {
    if (warp == K_WARP) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&sy->once, groups * TILE);
        for (int x = 0; x < groups; ++x)
          tma_load_3d(sm + x * TILE, &qmap, 0, g * GROUP, qbeg + q0 + x * QT, &sy->once);
      }
      load_tiles<PAGE, KS>(p, sp, &kmap, p.k, kring, sy->kfull, sy->kempty, list0, g, lane, abort);
      if (lane == 0) mbar_wait(&sy->once, 0, p.err);
    } else if (warp == V_WARP) {
      load_tiles<PAGE, VS>(p, sp, &vmap, p.v, vring, sy->vfull, sy->vempty, list0, g, lane, abort);
    } else if (warp == S_WARP) {
      const uint64_t qdesc = sw128_desc(qtile), kdesc = sw128_desc(smem_addr(kring));
      bool ok = warp_wait_quiet(&sy->once, 0, p.err, abort, lane);
      int t = 0;
      for (; t < ntiles && ok; ++t) {
        const int s = t % KS;
        ok = warp_wait_quiet(&sy->kfull[s], (t / KS) & 1, p.err, abort, lane);
        const uint64_t kd = kdesc + static_cast<uint64_t>(s * (TILE >> 4));
        for (int x = 0; x < groups && ok; ++x) {
          ok = t == 0 || warp_wait_quiet(&sy->sempty[x], (t - 1) & 1, p.err, abort, lane);
          if (!ok) break;
          tc_fence_after();
          if (lane == 0) {
            const uint64_t qd = qdesc + static_cast<uint64_t>(x * (TILE >> 4));
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) tc_mma(tmem + x * TMEM_TILE, qd + 2 * kk, kd + 2 * kk, IDESC_S, kk > 0);
            tc_commit(&sy->sfull[x]);
            if (x + 1 == groups) tc_commit(&sy->kempty[s]);
          }
        }
      }
      if (lane == 0) {
        if (!ok) *abort = 1;
        tc_commit(&sy->s_done);   // every product completes before the tensor memory may be freed
        mbar_wait(&sy->s_done, 0, p.err);
      }
    } else {
      const uint64_t vdesc = sw128_mn_desc(smem_addr(vring));
      bool ok = true;
      for (int t = 0; t < ntiles && ok; ++t) {
        const int s = t % VS;
        ok = warp_wait_quiet(&sy->vfull[s], (t / VS) & 1, p.err, abort, lane);
        if (!ok) break;
        if (!sp.whole(sp.key(t))) clean_values(sp, vring + s * TILE, sp.key(t), sy, lane);
        const uint64_t vd = vdesc + static_cast<uint64_t>(s * (TILE >> 4));
        for (int x = 0; x < groups && ok; ++x) {
          ok = warp_wait_quiet(&sy->pfull[x], t & 1, p.err, abort, lane);
          if (!ok) break;
          tc_fence_after();
          if (lane == 0) {
            const uint32_t base = tmem + x * TMEM_TILE;
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk)
              tc_mma_ts(base + O_COL, base + P_COL + kk * 8, vd + kk * (2048 >> 4), IDESC_PV, t > 0 || kk > 0);
            tc_commit(&sy->pempty[x]);
            if (x + 1 == groups) tc_commit(&sy->vempty[s]);
          }
        }
      }
      if (lane == 0) {
        if (ok) {
          mbar_arrive(&sy->odone);
          tc_commit(&sy->odone);
        } else {
          *abort = 1;
        }
        tc_commit(&sy->pv_done);
        mbar_wait(&sy->pv_done, 0, p.err);
      }
    }
    __syncwarp();
  } else if (warp / SM_WARPS < groups) {
    const int tile = warp / SM_WARPS, quarter = warp & 3, half = (warp >> 2) & 1;
    const int r = quarter * 32 + lane;           // accumulator row = TMEM lane
    const int q = q0 + tile * QT + r / GROUP;
    const int h = g * GROUP + r % GROUP;
    const int pos = prefix + min(q, nq - 1);
    const uint32_t lanes = tmem + tile * TMEM_TILE + (static_cast<uint32_t>(quarter * 32) << 16);
    // the positions of this warp's rows: a key tile that all of them see in
    // full needs no mask, whatever the CTA's other rows see
    Span own = sp;
    own.p_lo = prefix + min(q0 + tile * QT + quarter * 4, nq - 1);
    own.p_hi = prefix + min(q0 + tile * QT + quarter * 4 + 3, nq - 1);
    float (&top)[2][2][BM] = sy->top[tile];
    float m = -INFINITY, l = 0.f;
    if (groups == 2 && tile == 1) turn_give(0);   // tile 0 begins
    bool ok = true;   // after a timeout a warp only keeps its partner's barriers
    for (int t = 0; t < ntiles; ++t) {
      ok = ok && warp_wait_quiet(&sy->sfull[tile], t & 1, p.err, abort, lane);
      float mt = -INFINITY;
      const int k0 = sp.key(t);
      const bool edge = !own.whole(k0);
      const uint32_t scol = lanes + half * HALF;
      // keys of this thread's half that its row sees: i <= hi and (i > lo or i < fi)
      const int hi = pos - k0 - half * HALF, fi = sp.first - k0 - half * HALF;
      const int lo = sp.window < 0 || hi < 0 ? -1 : hi - sp.window;
      // The logits are read twice, 32 at a time, rather than kept: 64 of them do
      // not fit beside the rest in the 96 registers of a thread among 640.
      auto logits = [&](int c, float (&v)[32]) {
        __syncwarp();
        tmem_ld32(scol + c, v);
        if (edge) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = (c + i <= hi && (c + i > lo || c + i < fi)) ? v[i] : -INFINITY;
        }
      };
      if (ok) {
        tc_fence_after();
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < HALF; c += 32) {
          float v[32];
          logits(c, v);
#pragma unroll
          for (int i = 0; i < 32; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], v[i + 2 * k], v[i + 2 * k + 1]);
        }
        mt = p.scale2 * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        top[t & 1][half][r] = mt;
      }
      quarter_sync(tile * 4 + quarter);
      ok = ok && (t == 0 || warp_wait_quiet(&sy->pempty[tile], (t - 1) & 1, p.err, abort, lane));
      if (groups == 2) turn_wait(tile);
      if (!ok) {
        if (groups == 2 && (tile == 0 || t + 1 < ntiles)) turn_give(tile ^ 1);
        continue;
      }
      mt = fmaxf(mt, top[t & 1][half ^ 1][r]);
      tc_fence_after();
      const bool grow = mt > m + LAZY || (m == -INFINITY && mt > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float mn = grow ? mt : m;
        const float a = m == -INFINITY ? 0.f : fast_exp2(m - mn);
        l *= a;
        m = mn;
        if (t >= 1) {   // P V(t - 1) has completed: O is at rest; each half takes 32 of its columns
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 32; c += 8) {   // a few columns at a time: the tile's logits stay in registers
            float o[8];
            tmem_ld8(lanes + O_COL + half * 32 + c, o);
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(o[i] * a);
            tmem_st8_async(lanes + O_COL + half * 32 + c, w);
          }
        }
      }
      const float mu = m == -INFINITY ? 0.f : m;
      const uint32_t pcol = lanes + P_COL + half * (HALF / 2);
#pragma unroll
      for (int c = 0; c < HALF; c += 32) {
        float v[32];
        logits(c, v);
        if (c + 32 == HALF) {   // S is read: the next product may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sy->sempty[tile]);
        }
        l += weights(v, p.scale2, mu, pcol + c / 2);
      }
      if (groups == 2 && (tile == 0 || t + 1 < ntiles)) turn_give(tile ^ 1);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sy->pfull[tile]);
    }
    if (!ok) *abort = 1;
    top[ntiles & 1][half][r] = l;
    quarter_sync(tile * 4 + quarter);
    if (ok && warp_wait_quiet(&sy->odone, 0, p.err, abort, lane)) {
      l += top[ntiles & 1][half ^ 1][r];
      tc_fence_after();
      float o[32];
      __syncwarp();
      tmem_ld32(lanes + O_COL + half * 32, o);
      if (p.sinks) l += exp2f(p.sinks[h] * LOG2E - m);
      float f = 1.f / l;
      for (int e = 0; e < min(sy->edges, MAX_EDGE); ++e)
        for (int w = 0; w < 4; ++w)
          for (uint32_t bad = sy->edge_bad[e][w]; bad; bad &= bad - 1)
            if (sp.sees(pos, sy->edge_key[e] + w * 32 + __ffs(bad) - 1)) f = __int_as_float(0x7fc00000);
      if (q < nq) {
        uint4* dst = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(qbeg + q) * p.o_st +
                                              static_cast<int64_t>(h) * p.o_sh + half * 32);
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
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
  if (warp == S_WARP) tmem_dealloc(tmem, TMEM_COLS);
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
  if (!host::set_smem(attend_kernel<16>, SMEM) || !host::set_smem(attend_kernel<0>, SMEM))
    return host::fail(CE_ERR_CUDA, "ce_window_prefill: smem attr");
  const dim3 grid((max_q + TILES * QT - 1) / (TILES * QT), num_kv_heads, bs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (page_size == 16) attend_kernel<16><<<grid, THREADS, SMEM, st>>>(p, qmap, kmap, vmap);
  else attend_kernel<0><<<grid, THREADS, SMEM, st>>>(p, qmap, kmap, vmap);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_window_prefill launch");
  return CE_OK;
}
