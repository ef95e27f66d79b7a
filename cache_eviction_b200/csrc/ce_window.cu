// ce_window_prefill: causal attention of extend chunks with a sliding window
// and a few first tokens, over the paged bf16 pools, on the 5th-generation
// tensor cores.
//
//   out_i = softmax over {t <= p, t > p - window or t < first} (and the sink) of
//           scale q_i . k_t,  times v_t,    p = kv_tokens - nq + i
//
// An item is (32 queries, KV head, entry): two tiles of 16 queries whose 8 heads
// are a tile's 128 accumulator rows and share every key and value tile.  One
// CTA per SM takes every gridDim-th item, the last queries (which see the most
// keys) first, and walks the 128-key tiles that hold a visible token of some
// row (the first tokens' tiles, then the window's, which start at a page
// boundary), in one pass:
//   load warp     picks the items; queries through two slots of 32 KB, key and
//                 value tiles each through a ring of 16 KB slots (page loads by
//                 TMA, or cp.async gathers for pages under 8 tokens), page
//                 indices read a tile ahead
//   S warp        S(t) = Q K^T of both query tiles into tensor memory, each as
//                 soon as its S(t-1) is read
//   clean warp    value tiles that are seen in part made safe (below)
//   PV warp       O += P(t) V(t) of each once its weights are in place
//   softmax warps eight per query tile, two threads per row, 64 keys each: S from
//                 tensor memory, running maximum (exchanged through shared
//                 memory) and sum, P = 2^(s - m) in bf16 back into tensor
//                 memory as the A operand of the second product.  O is
//                 rescaled only when a row's maximum has grown by more than
//                 2^8 since the last rescale (P stays below 2^8, its relative
//                 precision and the fp32 sum's are the same).
// The warps go from item to item by themselves, through a ring of item slots:
// an item's loads, first products and clean-up run under the one before.  (A CTA
// per item left the SM idle while it started and ended: 207 us instead of 123
// for prompts of 4,093 and 3,069 tokens, 64 heads, window 128, where an item
// has two key tiles; 110 with the clean warp's loop rolled, 112 with a scale per
// row for large logits.)
// The exponentials bound long items (one per row and key on a unit of 16 per
// clock and SM: 2,048 clocks per key tile and item, against 1,536 of the tensor
// cores), so the two query tiles take turns at them: while one computes its
// weights the other's waits, reads and maxima go on.  Left to themselves (two
// CTAs per SM) the tiles fell into step, both at the exponentials and then both
// waiting.  2,048 queries behind 26,624 tokens (2,048 first + 6,144 window), 64
// heads: 504 us, 545 TFLOP/s, ~3,700 clocks per key tile and item; its 512
// items are 3.5 rounds of 148.  Short items are bound by their chain of waits
// (last product, normaliser, output, then the next item's first maximum).
// (Taking a share of the exponentials as a polynomial on the FMA pipes was
// slower at every share.  So was making a tile's weights with the maximum so
// far, finding its own beside them, 624 us: the maxima cost little while the
// product before is still running.)  P in bf16 is rounded by at most 2^-8 of
// itself, as the output is; over a row's keys these errors average out, to 5.9e-4
// (relative norm) for the prompts above and 1.8e-4 for the 2,048 queries, against
// 1.7e-3 for the output's rounding.  (The decode kernel splits P in two, which
// here would double the second product.)  Maxima, sums and O are fp32.
//
// What a row must not see must not reach it: a masked key's logit is replaced
// before the maximum, and a masked value meets P = 0, which is no help if it
// is infinite or NaN.  So in a tile that some row sees only in part the clean
// warp clears the values that no row sees (a page's unwritten slots, pages that
// were not loaded) and any value that is not finite, noting its token; a row
// that does see such a token gets NaN at the end.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

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
constexpr int KS = 4, VS = 4;            // ring slots of K and V tiles
constexpr int QS = 2;                    // items whose queries are in shared memory
constexpr int IS = 4;                    // items between the load warp and the last one to finish with one
constexpr int LAG = 3;                   // cp.async tiles in flight before one is published
constexpr int SM_WARPS = 8;              // softmax, per query tile: TMEM lanes 32 (w % 4) .. +31, keys 64 (w / 4) .. +63
constexpr int HALF = BN / 2;             // keys of a softmax thread
constexpr int L_WARP = TILES * SM_WARPS, C_WARP = L_WARP + 1, S_WARP = L_WARP + 2;   // load, clean, S and the PV warp
constexpr int THREADS = 32 * (TILES * SM_WARPS + 4);   // (one warp more would leave a thread 80 registers)
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
  int64_t items, whole;   // query tile pairs x KV heads x entries; from `whole` on single tiles
  int bs, xs;             // entries, query tile pairs of the longest one
  int total_q, max_q, max_tokens;
  int window, first;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  int32_t* err;
};

// One (32 or 16 queries, KV head, entry).
struct Item {
  int64_t number;                 // p.items: no more of them
  int g, q0, nq, prefix, qbeg, list0;   // queries q0 .. nq - 1, at most 32
};
struct ItemSlot : Item {
  int edges;                      // tiles in whose values the clean warp found some that are not finite
  int edge_key[MAX_EDGE];         // their first token
  uint32_t edge_bad[MAX_EDGE][4]; // their tokens with such a value
};

struct Sync {
  uint64_t kfull[KS], kempty[KS], vfull[VS], vclean[VS], vempty[VS], qfull[QS], qempty[QS], ifull[IS], iempty[IS];
  uint64_t sfull[TILES], sempty[TILES], pfull[TILES], pempty[TILES], odone[TILES];
  uint64_t s_done, pv_done;
  uint32_t tmem;
  int abort;
  ItemSlot items[IS];
  float top[TILES][2][2][BM];     // by query tile, key tile parity and half: the rows' maxima
  float sum[TILES][2][BM];        // and at the end of an item their sums
};

// The keys an item's rows (positions p_lo .. p_hi) see, as 128-key tiles.
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

// Item `number`, if its entry's ranges fit and it has a query.  The last
// queries, which see the most keys, come first.
__device__ __forceinline__ bool make_item(const Params& p, int64_t number, Item& it) {
  if (number >= p.items) return false;
  const int64_t per = static_cast<int64_t>(p.G) * p.bs;
  const bool single = number >= p.whole;
  const int64_t pair = single ? p.whole + (number - p.whole) / 2 : number;
  const int x = p.xs - 1 - static_cast<int>(pair / per);
  const int64_t gb = pair % per;
  const int b = static_cast<int>(gb / p.G);
  it.number = number;
  it.g = static_cast<int>(gb % p.G);
  it.q0 = x * (TILES * QT) + (single ? static_cast<int>((number - p.whole) & 1) * QT : 0);
  it.qbeg = p.qo_indptr[b];
  it.nq = p.qo_indptr[b + 1] - it.qbeg;
  it.list0 = p.kv_indptr[b];
  const int ntok = p.kv_tokens[b], pages = p.kv_indptr[b + 1] - it.list0;
  it.prefix = ntok - it.nq;
  const int64_t units = (static_cast<int64_t>(ntok) + p.P - 1) / p.P;
  const bool ok = it.qbeg >= 0 && it.nq >= 0 && it.qbeg + static_cast<int64_t>(it.nq) <= p.total_q && it.nq <= p.max_q &&
                  ntok <= p.max_tokens && ntok >= it.nq && it.list0 >= 0 && it.list0 + units <= p.kv_capacity &&
                  units <= pages;
  if (!ok && x == 0) flag_error(p.err, CE_EW_SHAPE);
  const bool some = ok && it.q0 < it.nq;
  it.nq = min(it.nq, it.q0 + (single ? QT : TILES * QT));
  return some;
}
__device__ __forceinline__ int groups_of(const Item& it) { return it.nq - it.q0 > QT ? 2 : 1; }   // query tiles with a query
__device__ __forceinline__ Span span_of(const Params& p, const Item& it) {
  return Span(p, it.prefix + it.q0, it.prefix + it.nq - 1);
}

// A position in a ring of n slots and the parity of its round.  (A wait for the
// parity before the first, 1, is over at once: the slots are empty.)
struct Ring {
  int slot = 0, n;
  uint32_t phase = 0;
  __device__ __forceinline__ explicit Ring(int slots) : n(slots) {}
  __device__ __forceinline__ void next() {
    if (++slot == n) {
      slot = 0;
      phase ^= 1;
    }
  }
};

// The i-th item of this CTA from its slot.  False: no more, or a wait gave up.
__device__ __forceinline__ bool next_item(const Params& p, Sync* sy, int i, Item& it, bool& ok, int lane) {
  ok = ok && warp_wait_quiet(&sy->ifull[i % IS], (i / IS) & 1, p.err, &sy->abort, lane);
  if (!ok) return false;
  __syncwarp();
  it = sy->items[i % IS];
  return it.number < p.items;
}
// Its slot may be used again (as far as this warp is concerned).
__device__ __forceinline__ void release_item(Sync* sy, int i, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(&sy->iempty[i % IS]);
}

// Where the load warp puts the tiles.
struct Rings {
  uint8_t *ktile, *vtile;
  uint64_t *kfull, *kempty, *vfull, *vempty;
  Ring k, v;
};

// The key and value tiles of one item into their rings; false once a wait gave
// up.  PAGE: tokens per page, or 0 for any size that divides 64.
template <int PAGE>
__device__ __forceinline__ bool load_tiles(const Params& p, const Span& sp, Rings& at, const CUtensorMap* kmap,
                                           const CUtensorMap* vmap, int list0, int g, int lane, volatile int* abort) {
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
  auto empty = [&](uint64_t* bars, const Ring& r) { return warp_wait_quiet(&bars[r.slot], r.phase ^ 1, p.err, abort, lane); };
  if (tma) {
    const int pages = BN / P;
    int next = lane < pages ? unit_of(sp.key(0) + lane * P) : -1;
    for (int t = 0; t < sp.ntiles; ++t) {
      const int k0 = sp.key(t) + lane * P;
      const int unit = lane < pages ? checked(next, k0) : -1;
      if (t + 1 < sp.ntiles) next = lane < pages ? unit_of(sp.key(t + 1) + lane * P) : -1;
      const int bytes = __popc(__ballot_sync(0xffffffffu, unit >= 0)) * P * 128, row = (unit * p.G + g) * P;
      if (!empty(at.kempty, at.k)) return false;
      if (lane == 0) mbar_arrive_expect_tx(&at.kfull[at.k.slot], bytes);
      __syncwarp();
      if (unit >= 0) tma_load_2d(at.ktile + at.k.slot * TILE + lane * P * 128, kmap, 0, row, &at.kfull[at.k.slot]);
      at.k.next();
      if (!empty(at.vempty, at.v)) return false;
      if (lane == 0) mbar_arrive_expect_tx(&at.vfull[at.v.slot], bytes);
      __syncwarp();
      if (unit >= 0) tma_load_2d(at.vtile + at.v.slot * TILE + lane * P * 128, vmap, 0, row, &at.vfull[at.v.slot]);
      at.v.next();
    }
    return true;
  }
  if constexpr (PAGE == 0) {
    auto publish = [&](int back) {   // the tile so many before the last
      if (lane == 0) {
        mbar_arrive(&at.kfull[(at.k.slot + KS - 1 - back) % KS]);
        mbar_arrive(&at.vfull[(at.v.slot + VS - 1 - back) % VS]);
      }
    };
    bool ok = true;
    int t = 0;
    for (; t < sp.ntiles; ++t) {
      const int k0 = sp.key(t);
      int u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = unit_of(k0 + lane + 32 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = checked(u[i], k0 + lane + 32 * i);
      ok = empty(at.kempty, at.k) && empty(at.vempty, at.v);
      if (!ok) break;
      const uint32_t kto = smem_addr(at.ktile) + at.k.slot * TILE, vto = smem_addr(at.vtile) + at.v.slot * TILE;
      const int c = lane & 7;
#pragma unroll 4
      for (int j = 0; j < BN / 4; ++j) {
        const int r = (lane >> 3) + 4 * j;
        const int from = (j >> 3) == 0 ? u[0] : (j >> 3) == 1 ? u[1] : (j >> 3) == 2 ? u[2] : u[3];
        const int unit = __shfl_sync(0xffffffffu, from, r & 31);
        const bool have = unit >= 0;   // rows that no query sees are zeros
        const int64_t off = have ? ((static_cast<int64_t>(unit) * p.G + g) * P + (k0 + r) % P) * D + c * 8 : 0;
        cp_async16(kto + swz(r, c), p.k + off, have);
        cp_async16(vto + swz(r, c), p.v + off, have);
      }
      at.k.next();
      at.v.next();
      cp_async_commit();
      if (t >= LAG) {
        cp_async_wait<LAG>();
        fence_proxy_async();
        __syncwarp();
        publish(LAG);
      }
    }
    cp_async_wait<0>();   // an item's tiles are all published before the next one's
    fence_proxy_async();
    __syncwarp();
    if (ok)
      for (int back = min(t, LAG) - 1; back >= 0; --back) publish(back);
    return ok;
  }
  return true;
}
// Every TMA load issued lands before the CTA may exit: the last round of each slot.
__device__ __forceinline__ void drain(uint64_t* full, Ring at, int32_t* err) {
  for (int s = 0; s < at.n; ++s) mbar_wait(&full[s], at.phase ^ (s >= at.slot ? 1u : 0u), err);
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
__device__ __forceinline__ void clean_values(const Span& sp, uint8_t* tile, int k, ItemSlot* it, int lane) {
  const int e = it->edges;
  __syncwarp();
  uint8_t* mine = tile + (lane >> 3) * 128 + (lane & 7) * 16;
  const int row0 = lane >> 3, end = sp.p_hi + 1 - k, from = sp.lo - k, head = sp.first - k;
  uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1   // (unrolled it took 9 % of the whole kernel: its instructions evict the softmax warps')
  for (int i0 = 0; i0 < BN / 4; i0 += 4) {
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint4*>(mine + (i0 + i) * 512);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
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
#pragma unroll 1
    for (int w = 0; w < 4; ++w) {
      uint32_t bad = 0u;
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        uint4* at = reinterpret_cast<uint4*>(mine + (w * 32 + i * 4) * 128);
        const uint4 x = *at;
        const uint4 nf = make_uint4(not_finite(x.x), not_finite(x.y), not_finite(x.z), not_finite(x.w));
        if (nf.x | nf.y | nf.z | nf.w) {
          *at = make_uint4(x.x & ~nf.x, x.y & ~nf.y, x.z & ~nf.z, x.w & ~nf.w);
          bad |= 1u << (i * 4 + (lane >> 3));
        }
      }
      bad = __reduce_or_sync(0xffffffffu, bad);
      if (lane == 0 && e < MAX_EDGE) it->edge_bad[e][w] = bad;
    }
    if (lane == 0 && e < MAX_EDGE) {
      it->edge_key[e] = k;
      it->edges = e + 1;
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

// A weight's exponent, scale2 v - m, is one rounding of the exact product, so at
// the maximum it is what m was rounded by: from 2^30 on that could leave fp32.
// There a row's scale is cut by a power of two that keeps m below 2^30: logits
// that differ at all differ by 32 octaves still.  Old and new maximum m and mt
// (in units of the scale so far) and the scale for a maximum that rises to mt.
constexpr float FAR = 1073741824.f;
__device__ __forceinline__ void rescale(float& m, float& mt, float& scale2, float full) {
  const float cut = full / scale2, now = mt * cut;   // in log2 units
  const int over = max(0, static_cast<int>(__float_as_uint(fabsf(now)) >> 23) - (127 + 29));
  const float by = __uint_as_float(static_cast<uint32_t>(127 - over) << 23);
  m = fmaxf(m * cut * by, now * by - FAR);           // (no further below than what makes a factor 0)
  mt = now * by;
  scale2 = full * by;
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

// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : 0xffffffffu >> (32 - min(n, 32)); }

constexpr int SMEM = 1024 + (QS * TILES + KS + VS) * TILE + static_cast<int>(sizeof(Sync));
// One CTA per SM (it holds all 512 TMEM columns): tcgen05.alloc never waits.
static_assert(SMEM <= 227 * 1024 && 2 * SMEM > 228 * 1024, "one CTA per SM");

template <int PAGE>
__global__ void __launch_bounds__(THREADS, 1)
    attend_kernel(const Params p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  const uint32_t qtile = smem_addr(sm);
  uint8_t *kring = sm + QS * TILES * TILE, *vring = kring + KS * TILE;
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
      mbar_init(&sy->vclean[i], 1);
      mbar_init(&sy->vempty[i], 1);
    }
    for (int i = 0; i < QS; ++i) {
      mbar_init(&sy->qfull[i], 1);
      mbar_init(&sy->qempty[i], 1);
    }
    for (int i = 0; i < IS; ++i) {
      mbar_init(&sy->ifull[i], 1);
      mbar_init(&sy->iempty[i], THREADS / 32 - 1);   // every warp but the load warp
    }
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&sy->sfull[i], 1);
      mbar_init(&sy->sempty[i], SM_WARPS);
      mbar_init(&sy->pfull[i], SM_WARPS);
      mbar_init(&sy->pempty[i], 1);
      mbar_init(&sy->odone[i], 2);   // an item's last product and the PV thread (the clean warp's notes are in place)
    }
    mbar_init(&sy->s_done, 1);
    mbar_init(&sy->pv_done, 1);
    sy->abort = 0;
    fence_mbar_init();
  }
  if (warp == S_WARP) tmem_alloc(&sy->tmem, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sy->tmem;

  if (warp >= L_WARP) {
    bool ok = true;
    Item it;
    if (warp == L_WARP) {
      // Chooses this CTA's items (blockIdx.x, + gridDim.x, ...; 32 looked at at a
      // time) and loads their queries, keys and values.
      Rings at{kring, vring, sy->kfull, sy->kempty, sy->vfull, sy->vempty, Ring(KS), Ring(VS)};
      Ring qat(QS);
      int64_t base = blockIdx.x;
      unsigned found = 0;
      for (int i = 0;; ++i) {
        while (!found && base < p.items) {
          found = __ballot_sync(0xffffffffu, make_item(p, base + static_cast<int64_t>(lane) * gridDim.x, it));
          base += 32LL * gridDim.x;
        }
        const int from = max(0, __ffs(static_cast<int>(found)) - 1);
        Item now;
        now.number = found ? __shfl_sync(0xffffffffu, it.number, from) : p.items;
        now.g = __shfl_sync(0xffffffffu, it.g, from);
        now.q0 = __shfl_sync(0xffffffffu, it.q0, from);
        now.nq = __shfl_sync(0xffffffffu, it.nq, from);
        now.prefix = __shfl_sync(0xffffffffu, it.prefix, from);
        now.qbeg = __shfl_sync(0xffffffffu, it.qbeg, from);
        now.list0 = __shfl_sync(0xffffffffu, it.list0, from);
        const int s = i % IS, qs = qat.slot;
        ok = warp_wait_quiet(&sy->iempty[s], ((i / IS) & 1) ^ 1, p.err, abort, lane);
        if (!ok) break;
        if (lane == 0) {
          static_cast<Item&>(sy->items[s]) = now;
          sy->items[s].edges = 0;
          mbar_arrive(&sy->ifull[s]);
        }
        if (!found) break;
        found &= found - 1;
        ok = warp_wait_quiet(&sy->qempty[qs], qat.phase ^ 1, p.err, abort, lane);
        if (!ok) break;
        qat.next();
        if (lane == 0) {
          const int groups = groups_of(now);
          mbar_arrive_expect_tx(&sy->qfull[qs], groups * TILE);
          for (int x = 0; x < groups; ++x)
            tma_load_3d(sm + (qs * TILES + x) * TILE, &qmap, 0, now.g * GROUP, now.qbeg + now.q0 + x * QT, &sy->qfull[qs]);
        }
        __syncwarp();
        ok = load_tiles<PAGE>(p, span_of(p, now), at, &kmap, &vmap, now.list0, now.g, lane, abort);
        if (!ok) break;
      }
      if (!ok) *abort = 1;
      if (lane == 0) {
        if (PAGE || p.P >= 8) {
          drain(sy->kfull, at.k, p.err);
          drain(sy->vfull, at.v, p.err);
        }
        drain(sy->qfull, qat, p.err);
      }
    } else if (warp == S_WARP) {
      const uint64_t qdesc = sw128_desc(qtile), kdesc = sw128_desc(smem_addr(kring));
      Ring k(KS);
      uint32_t turn = 0;   // bit x: the parity of query tile x's products so far
      for (int i = 0; next_item(p, sy, i, it, ok, lane); ++i) {
        release_item(sy, i, lane);
        const int groups = groups_of(it), ntiles = span_of(p, it).ntiles, qs = i % QS;
        ok = warp_wait_quiet(&sy->qfull[qs], (i / QS) & 1, p.err, abort, lane);
        for (int t = 0; t < ntiles && ok; ++t, k.next()) {
          ok = warp_wait_quiet(&sy->kfull[k.slot], k.phase, p.err, abort, lane);
          const uint64_t kd = kdesc + static_cast<uint64_t>(k.slot * (TILE >> 4));
#pragma unroll 1   // (unrolled, here and below, the kernel took 14 % longer)
          for (int x = 0; x < groups && ok; ++x) {
            ok = warp_wait_quiet(&sy->sempty[x], ((turn >> x) & 1) ^ 1, p.err, abort, lane);
            if (!ok) break;
            turn ^= 1u << x;
            tc_fence_after();
            if (lane == 0) {
              const uint64_t qd = qdesc + static_cast<uint64_t>((qs * TILES + x) * (TILE >> 4));
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) tc_mma(tmem + x * TMEM_TILE, qd + 2 * kk, kd + 2 * kk, IDESC_S, kk > 0);
              tc_commit(&sy->sfull[x]);
              if (x + 1 == groups) {
                tc_commit(&sy->kempty[k.slot]);
                if (t + 1 == ntiles) tc_commit(&sy->qempty[qs]);
              }
            }
          }
        }
      }
      if (lane == 0) {
        if (!ok) *abort = 1;
        tc_commit(&sy->s_done);   // every product completes before the tensor memory may be freed
        mbar_wait(&sy->s_done, 0, p.err);
      }
    } else if (warp == C_WARP) {
      Ring v(VS);
      for (int i = 0; next_item(p, sy, i, it, ok, lane); ++i) {
        const Span sp = span_of(p, it);
        for (int t = 0; t < sp.ntiles && ok; ++t, v.next()) {
          ok = warp_wait_quiet(&sy->vfull[v.slot], v.phase, p.err, abort, lane);
          if (!ok) break;
          if (!sp.whole(sp.key(t))) clean_values(sp, vring + v.slot * TILE, sp.key(t), &sy->items[i % IS], lane);
          if (lane == 0) mbar_arrive(&sy->vclean[v.slot]);
        }
        if (ok) release_item(sy, i, lane);
      }
      if (!ok) *abort = 1;
    } else {
      const uint64_t vdesc = sw128_mn_desc(smem_addr(vring));
      Ring v(VS);
      uint32_t turn = 0;
      for (int i = 0; next_item(p, sy, i, it, ok, lane); ++i) {
        release_item(sy, i, lane);
        const int groups = groups_of(it), ntiles = span_of(p, it).ntiles;
        for (int t = 0; t < ntiles && ok; ++t, v.next()) {
          ok = warp_wait_quiet(&sy->vclean[v.slot], v.phase, p.err, abort, lane);
          const uint64_t vd = vdesc + static_cast<uint64_t>(v.slot * (TILE >> 4));
#pragma unroll 1
          for (int x = 0; x < groups && ok; ++x) {
            ok = warp_wait_quiet(&sy->pfull[x], (turn >> x) & 1, p.err, abort, lane);
            if (!ok) break;
            turn ^= 1u << x;
            tc_fence_after();
            if (lane == 0) {
              const uint32_t base = tmem + x * TMEM_TILE;
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)
                tc_mma_ts(base + O_COL, base + P_COL + kk * 8, vd + kk * (2048 >> 4), IDESC_PV, t > 0 || kk > 0);
              tc_commit(&sy->pempty[x]);
              if (x + 1 == groups) tc_commit(&sy->vempty[v.slot]);
              if (t + 1 == ntiles) {
                mbar_arrive(&sy->odone[x]);
                tc_commit(&sy->odone[x]);
              }
            }
          }
        }
      }
      if (lane == 0) {
        if (!ok) *abort = 1;
        tc_commit(&sy->pv_done);
        mbar_wait(&sy->pv_done, 0, p.err);
      }
    }
    __syncwarp();
  } else {
    const int tile = warp / SM_WARPS, quarter = warp & 3, half = (warp >> 2) & 1;
    const int r = quarter * 32 + lane;           // accumulator row = TMEM lane
    const uint32_t lanes = tmem + tile * TMEM_TILE + (static_cast<uint32_t>(quarter * 32) << 16);
    float (&top)[2][2][BM] = sy->top[tile];
    uint32_t n = 0, done = 0;                    // this query tile's key tiles and items so far
    bool ok = true;   // after a timeout a warp only keeps the others' barriers
    if (tile == 1) turn_give(0);                 // tile 0 begins
    Item it;
    it.number = static_cast<int64_t>(blockIdx.x) - gridDim.x;
    for (int i = 0;; ++i) {
      if (!next_item(p, sy, i, it, ok, lane)) {
        if (ok) break;
        // the items that are left, whose barriers the other warps may be at
        int64_t number = it.number + gridDim.x;
        while (number < p.items && !make_item(p, number, it)) number += gridDim.x;
        if (number >= p.items) break;
      }
      const int groups = groups_of(it);
      if (tile < groups) {
        const Span sp = span_of(p, it);
        const int ntiles = sp.ntiles;
        const int q = it.q0 + tile * QT + r / GROUP;
        const int pos = it.prefix + min(q, it.nq - 1);
        // the positions of this warp's rows: a key tile that all of them see in
        // full needs no mask, whatever the item's other rows see
        Span own = sp;
        own.p_lo = it.prefix + min(it.q0 + tile * QT + quarter * 4, it.nq - 1);
        own.p_hi = it.prefix + min(it.q0 + tile * QT + quarter * 4 + 3, it.nq - 1);
        float m = -INFINITY, l = 0.f, scale2 = p.scale2;
        for (int t = 0; t < ntiles; ++t, ++n) {
          ok = ok && warp_wait_quiet(&sy->sfull[tile], n & 1, p.err, abort, lane);
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
              const uint32_t see = below(hi + 1 - c) & (~below(lo + 1 - c) | below(fi - c));
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = see & (1u << i) ? v[i] : -INFINITY;
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
            mt = scale2 * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            top[n & 1][half][r] = mt;
          }
          quarter_sync(tile * 4 + quarter);
          ok = ok && warp_wait_quiet(&sy->pempty[tile], (n & 1) ^ 1, p.err, abort, lane);
          if (groups == 2) turn_wait(tile);
          if (!ok) {
            if (groups == 2) turn_give(tile ^ 1);
            continue;
          }
          mt = fmaxf(mt, top[n & 1][half ^ 1][r]);
          tc_fence_after();
          const bool grow = mt > m + LAZY || (m == -INFINITY && mt > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            if (grow && (fabsf(mt) >= FAR || scale2 != p.scale2)) rescale(m, mt, scale2, p.scale2);
            const float mn = grow ? mt : m;
            const float a = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            l *= a;
            m = mn;
            if (t >= 1) {   // P V(t - 1) has completed: O is at rest; each half takes 32 of its columns
              __syncwarp();
#pragma unroll 1
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
            l += weights(v, scale2, mu, pcol + c / 2);
          }
          if (groups == 2) turn_give(tile ^ 1);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sy->pfull[tile]);
        }
        // the normaliser, while the last product runs
        const int h = it.g * GROUP + r % GROUP;
        const float sink = p.sinks ? p.sinks[h] * LOG2E : -INFINITY;
        sy->sum[tile][half][r] = l;
        quarter_sync(tile * 4 + quarter);
        l += sy->sum[tile][half ^ 1][r];
        if (p.sinks) l += exp2f(sink - m * (p.scale2 / scale2));
        float f = 1.f / l;
        ok = ok && warp_wait_quiet(&sy->odone[tile], done & 1, p.err, abort, lane);
        ++done;
        if (ok) {
          tc_fence_after();
          float o[32];
          __syncwarp();
          tmem_ld32(lanes + O_COL + half * 32, o);
          const ItemSlot& notes = sy->items[i % IS];
          for (int e = 0; e < min(notes.edges, MAX_EDGE); ++e)
            for (int w = 0; w < 4; ++w)
              for (uint32_t bad = notes.edge_bad[e][w]; bad; bad &= bad - 1)
                if (sp.sees(pos, notes.edge_key[e] + w * 32 + __ffs(bad) - 1)) f = __int_as_float(0x7fc00000);
          if (q < it.nq) {
            uint4* dst = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(it.qbeg + q) * p.o_st +
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
      if (ok) release_item(sy, i, lane);
    }
    if (tile == 0) turn_wait(0);                 // the last turn given
    if (!ok) *abort = 1;
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
  p.bs = bs;
  p.xs = (max_q + TILES * QT - 1) / (TILES * QT);
  // A last round that would leave half of the SMs or more without an item is
  // given out as single query tiles, which take a CTA about 0.87 of a pair's time
  // (64 queries behind 26,624 tokens 132 -> 115 us, 256 of them 134 -> 119 us, the
  // chunk of the header, whose last round has 68 items, 542 -> 538 us, before the
  // clean warp's loop was rolled).
  const int sms = host::sm_count();
  p.items = static_cast<int64_t>(p.xs) * num_kv_heads * bs;
  p.whole = p.items;
  const int64_t rest = p.items % sms;
  if (2 * rest <= sms) {
    p.whole -= rest;
    p.items += rest;
  }
  p.total_q = total_q;
  p.max_q = max_q;
  p.max_tokens = max_tokens;
  p.window = window;
  p.first = first;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.err = err;
  if (host::window_prepare_device() != CE_OK) return CE_ERR_CUDA;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(p.items, sms));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (page_size == 16) attend_kernel<16><<<grid, THREADS, SMEM, st>>>(p, qmap, kmap, vmap);
  else attend_kernel<0><<<grid, THREADS, SMEM, st>>>(p, qmap, kmap, vmap);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_window_prefill launch");
  return CE_OK;
}

int ce::host::window_prepare_device() {
  if (!set_smem(window::attend_kernel<16>, window::SMEM) || !set_smem(window::attend_kernel<0>, window::SMEM))
    return fail_cuda("windowed prefill kernels: set-up");
  return CE_OK;
}
