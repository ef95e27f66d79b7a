// ce_kv4_write / ce_kv4_read: K and V rows quantised to 4 bits as they are
// written into the paged pools, and pages read back as bf16.  The page format
// and the rounding are in ce_kv4.cuh.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "ce_common.cuh"
#include "ce_host.h"
#include "ce_kv4.cuh"

namespace ce {
namespace kv4 {

constexpr int THREADS = 256;

struct WriteParams {
  const __nv_bfloat16* x[2];   // K, V rows
  int64_t st[2], sg[2];        // token and head strides (elements)
  uint8_t* pool[2];
  const int64_t* loc;
  int64_t tokens, pool_units;
  int G;
  int32_t* err;
};

constexpr float MAGIC = 12582912.f;   // 1.5 * 2^23: adding it rounds to integers, ties to even

// A code by definition: rint of the fp32 quotient d / s, at most 15.
__device__ __noinline__ uint32_t divide(float d, float s) {
  return static_cast<uint32_t>(fminf(rintf(__fdiv_rn(d, s)), 15.f));
}

// r = MAGIC + c with c off by at most one from rint(d / s): the remainder d - c s,
// which is exact (c s has 13 bits and d lies within a factor of two of it, or
// c is 0), tells on which side of the tie the quotient lies.  (The fp32
// quotient is a tie only where the exact one is: s has 8 bits.)
__device__ __forceinline__ uint32_t settle(float r, float d, float s) {
  const float e = fmaf(MAGIC - r, s, d), over = fabsf(e) - 0.5f * s;
  if (over > 0.f || (over == 0.f && (__float_as_uint(r) & 1u))) r += e > 0.f ? 1.f : -1.f;
  return __float_as_uint(fminf(r, MAGIC + 15.f));
}

// Codes of a lane's eight values (dims 8 l .. 8 l + 7) as bytes, four in a and
// four in b.  The product with an approximate reciprocal (2^-23) is within
// 15 * 2^-21 of the quotient, so it rounds to the same code unless it lies
// that close to a tie.  Rows whose span or reciprocal overflows divide.
__device__ __forceinline__ void encode(const uint32_t (&w)[4], float lo, float s, uint32_t& a, uint32_t& b) {
  a = b = 0u;
  if (!(s > 0.f)) return;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const uint64_t minus = pair(-lo, -lo), by = pair(inv, inv), magic = pair(MAGIC, MAGIC), back = pair(-MAGIC, -MAGIC);
  float off = 0.f;   // the largest distance from a code
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t t = mul2(add2(pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)), minus), by);
    const uint64_t m = add2(t, magic);
    float d0, d1, m0, m1;
    split(fma2(add2(m, back), pair(-1.f, -1.f), t), d0, d1);
    split(m, m0, m1);
    off = max3(off, fabsf(d0), fabsf(d1));
    r[2 * i] = __float_as_uint(m0);
    r[2 * i + 1] = __float_as_uint(m1);
  }
  if (s < 7.5e-37f || s > 2e37f) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = i < 4 ? (i < 2 ? w[0] : w[1]) : (i < 6 ? w[2] : w[3]);
      const float v = __uint_as_float((i & 1) ? x & 0xffff0000u : x << 16);
      // (halves of the large ones, exact, where the span lies beyond fp32's end)
      const uint32_t c = s > 1.f ? divide(v * 0.5f - lo * 0.5f, s * 0.5f) : divide(v - lo, s);
      if (i < 4) a |= c << (8 * i);
      else b |= c << (8 * i - 32);
    }
    return;
  }
  if (off > 0.49999f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[2 * i] = settle(__uint_as_float(r[2 * i]), __uint_as_float(w[i] << 16) - lo, s);
      r[2 * i + 1] = settle(__uint_as_float(r[2 * i + 1]), __uint_as_float(w[i] & 0xffff0000u) - lo, s);
    }
  }
  a = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
  b = __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410);
}

// A warp takes four consecutive tokens of one head, eight lanes per row, K and
// V in turn.  Tokens are counted so that a run of consecutive slots falls into
// aligned quads of a page (the first token's slot gives the phase); a whole
// quad's V bytes are gathered into words and stored as 128 consecutive bytes,
// any other set of slots byte by byte.  29,719 tokens of 8 heads take about
// 33 us (76 MB), 2.8 times what the bytes need: no unit is saturated (issue
// slots 70 %, ALU 62 %, 44 % of the warps), a warp waits for a quad's rows before
// it rounds, packs and exchanges their codes.
__global__ void __launch_bounds__(THREADS) write_kernel(const WriteParams p) {
  const int lane = threadIdx.x & 31, l = lane & 7, jq = lane >> 3;
  const int64_t first = p.loc[0];
  const int shift = first >= 0 ? static_cast<int>(first & 3) : 0;
  const int64_t quads = (p.tokens + shift + 3) / 4, warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
  const int g = blockIdx.y;
  for (int64_t quad = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); quad < quads;
       quad += warps) {
    const int64_t tok = quad * 4 + jq - shift;
    const int64_t loc = tok >= 0 && tok < p.tokens ? p.loc[tok] : -1;
    const int64_t unit = loc >= 0 ? loc / P : -1;
    const int j = static_cast<int>(loc & (P - 1));
    const bool ok = unit >= 0 && unit < p.pool_units;
    if (unit >= p.pool_units && l == 0) flag_error(p.err, CE_EW_INDEX);
    uint4 raw[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      raw[kv] = make_uint4(0, 0, 0, 0);
      if (ok) raw[kv] = *reinterpret_cast<const uint4*>(p.x[kv] + tok * p.st[kv] + g * p.sg[kv] + l * 8);
    }
    const int64_t loc0 = __shfl_sync(0xffffffffu, loc, 0);
    const bool whole = __all_sync(0xffffffffu, ok && (loc0 & 3) == 0 && loc == loc0 + jq);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint32_t w[4] = {raw[kv].x, raw[kv].y, raw[kv].z, raw[kv].w};
      // smallest and largest of the row; a NaN takes both
      auto b2 = [](uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
      __nv_bfloat162 mn = __hmin2_nan(__hmin2_nan(b2(w[0]), b2(w[1])), __hmin2_nan(b2(w[2]), b2(w[3])));
      __nv_bfloat162 mx = __hmax2_nan(__hmax2_nan(b2(w[0]), b2(w[1])), __hmax2_nan(b2(w[2]), b2(w[3])));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        mn = __hmin2_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = __hmax2_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
      const float lo = __bfloat162float(__hmin_nan(mn.x, mn.y)), hi = __bfloat162float(__hmax_nan(mx.x, mx.y));
      const bool finite = fabsf(lo) < INFINITY && fabsf(hi) < INFINITY;
      const __nv_bfloat16 sb = __float2bfloat16_rn((hi * 0.5f - lo * 0.5f) * (2.0f / 15.0f));
      uint32_t a, b;
      encode(w, lo, finite ? __bfloat162float(sb) : 0.f, a, b);
      uint8_t* slice = p.pool[kv] + (unit * p.G + g) * SLICE;
      if (kv == 0) {
        // bytes 2 i and 2 i + 1 into one: the even dim in the low half
        if (ok) *reinterpret_cast<uint32_t*>(slice + k_word(j, l)) = __byte_perm(a | (a >> 4), b | (b >> 4), 0x6420);
      } else {
        // V bytes pair dims r and r + 8 of a 16-dim block: lane h of the two that
        // share block q makes those of r = 4 h .. 4 h + 3
        const int q = l >> 1, h = l & 1;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, h ? a : b, 1);
        const uint32_t bytes = h ? got | (b << 4) : a | (got << 4);
        if (whole) {
          // 4 x 4 bytes across the tokens: lane jq ends with r = 4 h + jq of all four
          const uint32_t x = __shfl_xor_sync(0xffffffffu, bytes, 8);
          const uint32_t y = (jq & 1) ? __byte_perm(x, bytes, 0x7351) : __byte_perm(bytes, x, 0x6240);
          const uint32_t z = __shfl_xor_sync(0xffffffffu, y, 16);
          const uint32_t word = (jq & 2) ? __byte_perm(z, y, 0x7632) : __byte_perm(y, z, 0x5410);
          *reinterpret_cast<uint32_t*>(slice + v_byte(j & ~3, q, 4 * h + jq)) = word;
        } else if (ok) {
#pragma unroll
          for (int i = 0; i < 4; ++i) slice[v_byte(j, q, 4 * h + i)] = static_cast<uint8_t>(bytes >> (8 * i));
        }
      }
      if (l == 0 && ok) {
        const uint32_t sm = __bfloat16_as_ushort(sb), mm = __float_as_uint(lo) >> 16;
        *reinterpret_cast<uint32_t*>(slice + CODE_BYTES + j * 4) = finite ? (sm | (mm << 16)) : 0x7fc07fc0u;
      }
    }
  }
}

struct ReadParams {
  const uint8_t* pool[2];
  __nv_bfloat16* out[2];
  int64_t ou[2], og[2], ot[2];   // page, head and token strides of the outputs (elements)
  const int32_t* units;
  int64_t n, pool_units;
  int G;
  int32_t* err;
};

// Values m + c s of eight codes as four bf16 pairs.
__device__ __forceinline__ void decode8(uint32_t code, uint32_t par, uint32_t (&o)[4]) {
  const float s = __uint_as_float(par << 16), m = __uint_as_float(par & 0xffff0000u);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    // 2^23 + c in fp32 has c in its low bits
    const float a = __uint_as_float(((code >> (8 * d)) & 15u) | 0x4b000000u) - 8388608.f;
    const float b = __uint_as_float(((code >> (8 * d + 4)) & 15u) | 0x4b000000u) - 8388608.f;
    const __nv_bfloat162 v = __floats2bfloat162_rn(fmaf(a, s, m), fmaf(b, s, m));
    o[d] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

// One step of an 8 x 8 nibble transpose over eight lanes: swaps the halves of
// lanes that differ in bit `o` (nibbles that differ in the same bit).
template <int o, uint32_t KEEP>
__device__ __forceinline__ uint32_t swap_nibbles(uint32_t w, int n) {
  const uint32_t x = __shfl_xor_sync(0xffffffffu, w, o);
  return (n & o) ? (w & ~KEEP) | ((x >> (4 * o)) & KEEP) : (w & KEEP) | ((x << (4 * o)) & ~KEEP);
}

// One warp per (page, head), 16 coalesced bytes of codes per lane and operand.
//   K: lane (pair = lane / 4, t) holds dims 16 t .. of tokens 2 pair and 2 pair + 1.
//   V: lane (tg = lane / 8, r) holds, for each 16-dim block q, dims r and r + 8
//      of tokens 4 tg ..: after the transpose over r, lane (tg, n) holds eight
//      consecutive dims, 16 q + 8 (n % 2) .., of token 4 tg + n / 2.
// 4,096 pages of 8 heads (172 MB) take 34 us, 5.0 TB/s.
__global__ void __launch_bounds__(THREADS) read_kernel(const ReadParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
  const int g = blockIdx.y;
  for (int64_t pg = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); pg < p.n; pg += warps) {
    const int unit = p.units[pg];
    if (unit < 0 || unit >= p.pool_units) {
      if (unit >= 0 && lane == 0) flag_error(p.err, CE_EW_INDEX);
      continue;
    }
    const int64_t off = (static_cast<int64_t>(unit) * p.G + g) * SLICE;
    const uint8_t *ks = p.pool[0] + off, *vs = p.pool[1] + off;
    const int pair = lane >> 2, t = lane & 3, n = lane & 7, vt = (lane >> 3) * 4 + (n >> 1);
    const uint4 kc = *reinterpret_cast<const uint4*>(ks + lane * 16);
    const uint2 kp = *reinterpret_cast<const uint2*>(ks + CODE_BYTES + pair * 8);
    const uint4 vc = *reinterpret_cast<const uint4*>(vs + lane * 16);
    const uint32_t vp = *reinterpret_cast<const uint32_t*>(vs + CODE_BYTES + vt * 4);
    __nv_bfloat16* ko = p.out[0] + pg * p.ou[0] + g * p.og[0] + 2 * pair * p.ot[0] + t * 16;
    __nv_bfloat16* vo = p.out[1] + pg * p.ou[1] + g * p.og[1] + vt * p.ot[1] + (n & 1) * 8;
    uint32_t o[4];
    decode8(kc.x, kp.x, o);
    *reinterpret_cast<uint4*>(ko) = make_uint4(o[0], o[1], o[2], o[3]);
    decode8(kc.y, kp.x, o);
    *reinterpret_cast<uint4*>(ko + 8) = make_uint4(o[0], o[1], o[2], o[3]);
    decode8(kc.z, kp.y, o);
    *reinterpret_cast<uint4*>(ko + p.ot[0]) = make_uint4(o[0], o[1], o[2], o[3]);
    decode8(kc.w, kp.y, o);
    *reinterpret_cast<uint4*>(ko + p.ot[0] + 8) = make_uint4(o[0], o[1], o[2], o[3]);
    const uint32_t vw[4] = {vc.x, vc.y, vc.z, vc.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // nibble 2 j + half of lane r -> nibble r of lane 2 j + half
      uint32_t w = vw[q];
      w = swap_nibbles<4, 0x0000ffffu>(w, n);
      w = swap_nibbles<2, 0x00ff00ffu>(w, n);
      w = swap_nibbles<1, 0x0f0f0f0fu>(w, n);
      decode8(w, vp, o);
      *reinterpret_cast<uint4*>(vo + q * 16) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

}  // namespace kv4
}  // namespace ce

using namespace ce;

namespace {
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
}  // namespace

extern "C" int ce_kv4_write(const void* k, int64_t k_st, int64_t k_sg, const void* v, int64_t v_st, int64_t v_sg,
                            const int64_t* loc, int64_t tokens, int32_t num_kv_heads, int32_t head_dim,
                            int32_t page_size, void* k_pool, void* v_pool, int64_t pool_units, int32_t* err,
                            void* stream) {
  if (tokens < 0 || pool_units < 0 || num_kv_heads <= 0) return host::fail(CE_ERR_ARG, "ce_kv4_write: bad size");
  if (num_kv_heads > 65535) return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_write: more than 65535 heads");
  if (head_dim != kv4::D || page_size != kv4::P)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_write: needs head_dim 64 and 16-token pages");
  if (tokens == 0) return CE_OK;
  if (!k || !v || !loc || !k_pool || !v_pool) return host::fail(CE_ERR_ARG, "ce_kv4_write: null pointer");
  if ((k_st | k_sg | v_st | v_sg) % 8 || !aligned16(k) || !aligned16(v) || !aligned16(k_pool) || !aligned16(v_pool))
    return host::fail(CE_ERR_ARG, "ce_kv4_write: rows and pools need 16-byte alignment (strides multiples of 8)");
  const int sms = host::sm_count();
  if (sms <= 0) return host::fail(CE_ERR_CUDA, "no device");
  kv4::WriteParams p{};
  p.x[0] = static_cast<const __nv_bfloat16*>(k);
  p.x[1] = static_cast<const __nv_bfloat16*>(v);
  p.st[0] = k_st;
  p.st[1] = v_st;
  p.sg[0] = k_sg;
  p.sg[1] = v_sg;
  p.pool[0] = static_cast<uint8_t*>(k_pool);
  p.pool[1] = static_cast<uint8_t*>(v_pool);
  p.loc = loc;
  p.tokens = tokens;
  p.pool_units = pool_units;
  p.G = num_kv_heads;
  p.err = err;
  // a warp per quad of tokens (one more for the phase) and head, up to 16 blocks per SM
  const int64_t want = ((tokens + 6) / 4 + kv4::THREADS / 32 - 1) / (kv4::THREADS / 32);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(want, std::max(1, 16 * sms / num_kv_heads))), num_kv_heads);
  kv4::write_kernel<<<grid, kv4::THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_write launch");
  return CE_OK;
}

extern "C" int ce_kv4_read(const void* k_pool, const void* v_pool, int64_t pool_units, const int32_t* units,
                           int64_t num_units, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, void* k_out,
                           int64_t k_ou, int64_t k_og, int64_t k_ot, void* v_out, int64_t v_ou, int64_t v_og,
                           int64_t v_ot, int32_t* err, void* stream) {
  if (num_units < 0 || pool_units < 0 || num_kv_heads <= 0) return host::fail(CE_ERR_ARG, "ce_kv4_read: bad size");
  if (num_kv_heads > 65535) return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_read: more than 65535 heads");
  if (head_dim != kv4::D || page_size != kv4::P)
    return host::fail(CE_ERR_UNSUPPORTED, "ce_kv4_read: needs head_dim 64 and 16-token pages");
  if (num_units == 0) return CE_OK;
  if (!k_pool || !v_pool || !units || !k_out || !v_out) return host::fail(CE_ERR_ARG, "ce_kv4_read: null pointer");
  if ((k_ou | k_og | k_ot | v_ou | v_og | v_ot) % 8 || !aligned16(k_out) || !aligned16(v_out) || !aligned16(k_pool) ||
      !aligned16(v_pool))
    return host::fail(CE_ERR_ARG, "ce_kv4_read: outputs and pools need 16-byte alignment (strides multiples of 8)");
  const int sms = host::sm_count();
  if (sms <= 0) return host::fail(CE_ERR_CUDA, "no device");
  kv4::ReadParams p{};
  p.pool[0] = static_cast<const uint8_t*>(k_pool);
  p.pool[1] = static_cast<const uint8_t*>(v_pool);
  p.out[0] = static_cast<__nv_bfloat16*>(k_out);
  p.out[1] = static_cast<__nv_bfloat16*>(v_out);
  p.ou[0] = k_ou;
  p.ou[1] = v_ou;
  p.og[0] = k_og;
  p.og[1] = v_og;
  p.ot[0] = k_ot;
  p.ot[1] = v_ot;
  p.units = units;
  p.n = num_units;
  p.pool_units = pool_units;
  p.G = num_kv_heads;
  p.err = err;
  const int64_t want = (num_units + kv4::THREADS / 32 - 1) / (kv4::THREADS / 32);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(want, std::max(1, 16 * sms / num_kv_heads))), num_kv_heads);
  kv4::read_kernel<<<grid, kv4::THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_read launch");
  return CE_OK;
}

int ce::host::kv4_copy_prepare_device() {
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, kv4::write_kernel) != cudaSuccess ||
      cudaFuncGetAttributes(&a, kv4::read_kernel) != cudaSuccess)
    return host::fail_cuda("4-bit write and read kernels: set-up");
  return CE_OK;
}
