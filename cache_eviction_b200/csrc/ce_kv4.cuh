// The 4-bit page format of the KV cache, shared by ce_kv4.cu (write, read
// back) and ce_kv4_decode.cu (attention).
//
// A pool holds [units, G] slices of SLICE bytes, one per (unit, KV head): 16
// tokens of 64 values.  A token's row x is kept as 64 codes c in 0..15, a
// scale s and a minimum m, the value being m + c * s:
//   m = min(x)                 (exact: a bf16 input)
//   s = bf16((max / 2 - min / 2) * (2 / 15))      (halves, so that it cannot overflow)
//   c = clamp(rint((x - m) / s), 0, 15)           (fp32, ties to even; 0 where s is 0;
//                                                  by halves where x - m is beyond fp32)
// The scale's rounding to bf16 moves the top code by at most 15 * 2^-8 of a
// step.  A row that holds a NaN or an infinity is kept as s = m = NaN, c = 0.
//
// Bytes 0..511 are the codes, bytes 512 + 4 j .. the scale and then the
// minimum of token j.  The code order puts what one lane of the decode kernel
// needs for a page into one 16-byte load, already in the order of its
// m16n8k16 A fragments (lane = 4 r + t):
//   K  token j, dims 16 t .. 16 t + 15: the 8 bytes at ((j / 2) * 4 + t) * 16 +
//      (j % 2) * 8, dims in nibble order (low half first).  Lane (r, t) reads
//      tokens 2 r and 2 r + 1.
//   V  byte ((j / 4) * 8 + r) * 16 + q * 4 + j % 4 holds dims 16 q + r (low
//      half) and 16 q + r + 8 (high half) of token j.  Lane (r, t) reads
//      tokens 4 t .. 4 t + 3 of dims r and r + 8 of every 16-dim block q.
// Every byte belongs to one token, so that a token is written without reading
// its neighbours.
#pragma once

#include <cstdint>

namespace ce {
namespace kv4 {

constexpr int D = 64;
constexpr int P = 16;                       // tokens per page
constexpr int CODE_BYTES = P * D / 2;       // 512
constexpr int SLICE = CODE_BYTES + P * 4;   // 576

// Byte of the 8 K codes of token j, dims 8 l .. 8 l + 7 (one 32-bit word).
__host__ __device__ __forceinline__ int k_word(int j, int l) {
  return ((j >> 1) * 4 + (l >> 1)) * 16 + (j & 1) * 8 + (l & 1) * 4;
}
// Byte of dims 16 q + r and 16 q + r + 8 of token j in V.
__host__ __device__ __forceinline__ int v_byte(int j, int q, int r) {
  return ((j >> 2) * 8 + r) * 16 + q * 4 + (j & 3);
}

}  // namespace kv4
}  // namespace ce
