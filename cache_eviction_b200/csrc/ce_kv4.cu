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

// Eight lanes per (token, head) row, eight values each, K and V in turn.
__global__ void __launch_bounds__(THREADS) write_kernel(const WriteParams p) {
  const int l = threadIdx.x & 7;
  const int64_t rows = p.tokens * p.G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (THREADS / 8);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (THREADS / 8) + (threadIdx.x >> 3);
  const int64_t rounds = (rows + step - 1) / step;   // the same for every lane of a warp
  for (int64_t it = 0; it < rounds; ++it) {
    const int64_t row = first + it * step;
    const int64_t tok = row / p.G;
    const int g = static_cast<int>(row - tok * p.G);
    const bool in = row < rows;
    const int64_t loc = in ? p.loc[tok] : -1;
    const int64_t unit = loc >= 0 ? loc / P : -1;
    const int j = static_cast<int>(loc & (P - 1));
    const bool ok = unit >= 0 && unit < p.pool_units;
    if (unit >= p.pool_units && l == 0) flag_error(p.err, CE_EW_INDEX);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (ok) raw = *reinterpret_cast<const uint4*>(p.x[kv] + tok * p.st[kv] + g * p.sg[kv] + l * 8);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      float x[8];
      uint32_t mag = 0;   // largest bit pattern without signs: >= 0x7f80 means NaN or infinity
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        mag = max(mag, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
      }
      float lo = x[0], hi = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, o));
      }
      const bool finite = mag < 0x7f80u;
      const __nv_bfloat16 sb = __float2bfloat16_rn((hi * 0.5f - lo * 0.5f) * (2.0f / 15.0f));
      const float s = __bfloat162float(sb);
      uint32_t code = 0;
      if (finite && s > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = fminf(rintf(__fdiv_rn(x[i] - lo, s)), 15.f);
          code |= static_cast<uint32_t>(c) << (4 * i);
        }
      }
      // the other half of a 16-dim block: V bytes pair dims r and r + 8
      const uint32_t other = __shfl_xor_sync(0xffffffffu, code, 1);
      if (!ok) continue;
      uint8_t* slice = p.pool[kv] + (unit * p.G + g) * SLICE;
      if (kv == 0) {
        *reinterpret_cast<uint32_t*>(slice + k_word(j, l)) = code;
      } else {
        const int q = l >> 1, h = l & 1;
        const uint32_t lo4 = h ? other : code, hi4 = h ? code : other;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = h * 4 + i;
          slice[v_byte(j, q, r)] = static_cast<uint8_t>(((lo4 >> (4 * r)) & 15u) | (((hi4 >> (4 * r)) & 15u) << 4));
        }
      }
      if (l == 0) {
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

// One warp per (page, head): lane (tok = lane / 8, l = lane % 8) writes dims
// 8 l .. 8 l + 7 of tokens tok, tok + 4, ...
__global__ void __launch_bounds__(THREADS) read_kernel(const ReadParams p) {
  const int lane = threadIdx.x & 31, l = lane & 7;
  const int64_t items = p.n * p.G;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); it < items; it += warps) {
    const int64_t pg = it / p.G;
    const int g = static_cast<int>(it - pg * p.G);
    const int unit = p.units[pg];
    if (unit < 0 || unit >= p.pool_units) {
      if (unit >= 0 && lane == 0) flag_error(p.err, CE_EW_INDEX);
      continue;
    }
    const int64_t off = (static_cast<int64_t>(unit) * p.G + g) * SLICE;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint8_t* slice = p.pool[kv] + off;
      __nv_bfloat16* out = p.out[kv] + pg * p.ou[kv] + g * p.og[kv] + l * 8;
#pragma unroll
      for (int i = 0; i < P / 4; ++i) {
        const int j = (lane >> 3) + 4 * i;
        const uint32_t par = *reinterpret_cast<const uint32_t*>(slice + CODE_BYTES + j * 4);
        const float s = __uint_as_float(par << 16), m = __uint_as_float(par & 0xffff0000u);
        uint32_t code = 0;
        if (kv == 0) {
          code = *reinterpret_cast<const uint32_t*>(slice + k_word(j, l));
        } else {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            code |= ((static_cast<uint32_t>(slice[v_byte(j, l >> 1, r)]) >> (4 * (l & 1))) & 15u) << (4 * r);
        }
        uint32_t o[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const float a = fmaf(static_cast<float>((code >> (8 * d)) & 15u), s, m);
          const float b = fmaf(static_cast<float>((code >> (8 * d + 4)) & 15u), s, m);
          const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
          o[d] = *reinterpret_cast<const uint32_t*>(&v);
        }
        *reinterpret_cast<uint4*>(out + j * p.ot[kv]) = make_uint4(o[0], o[1], o[2], o[3]);
      }
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
  const int64_t want = (tokens * num_kv_heads + kv4::THREADS / 8 - 1) / (kv4::THREADS / 8);
  const int grid = static_cast<int>(std::min<int64_t>(want, 8LL * sms));
  kv4::write_kernel<<<grid, kv4::THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  if (cudaPeekAtLastError() != cudaSuccess) return host::fail_cuda("ce_kv4_write launch");
  return CE_OK;
}

extern "C" int ce_kv4_read(const void* k_pool, const void* v_pool, int64_t pool_units, const int32_t* units,
                           int64_t num_units, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, void* k_out,
                           int64_t k_ou, int64_t k_og, int64_t k_ot, void* v_out, int64_t v_ou, int64_t v_og,
                           int64_t v_ot, int32_t* err, void* stream) {
  if (num_units < 0 || pool_units < 0 || num_kv_heads <= 0) return host::fail(CE_ERR_ARG, "ce_kv4_read: bad size");
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
  const int64_t want = (num_units * num_kv_heads + kv4::THREADS / 32 - 1) / (kv4::THREADS / 32);
  const int grid = static_cast<int>(std::min<int64_t>(want, 8LL * sms));
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
