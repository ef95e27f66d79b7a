// Shared by the decode kernels (bf16 pages: ce_decode.cu, 4-bit pages:
// ce_kv4_decode.cu): the parameters of a decode call, the split of a batch
// into stages over CTAs and the workspace.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include "ce_common.cuh"
#include "ce_host.h"

namespace ce {
namespace decode {

constexpr int D = 64;
constexpr int GROUP = 8;
constexpr int NCW = 8;                    // consumer warps
constexpr int REC_ROWS = NCW * 8;         // virtual rows: warp w, head-row r
constexpr int REC_FLOATS = REC_ROWS * D + 2 * REC_ROWS;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Params {
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_tokens;
  int64_t kv_capacity;
  int64_t pool_units;
  const float* sinks;
  const int32_t* mode_of_row;
  const int64_t* rows;
  float scale_log2;
  int bs, H, G;
  float* scores;
  int64_t score_sg;
  int zero_new;
  void* out;
  int out_f32;
  int64_t o_sb, o_sh;
  float* lse_out;
  int32_t* prefix;   // [bs + 1] stage prefix (written by CTA 0)
  float* lse2;       // [bs, H] log2 normaliser per query head (for scores)
  float* rec;        // [(bs + grid), REC_FLOATS]
  float* ul;         // [kv_capacity, H] unit log-mass (log2 units) or null
  float* tl;         // [kv_capacity * P, H] token logits (page_size > 1, MAX rows) or null
  int window, first; // windowed decode: tokens t >= n - window or t < first (window < 0: all)
  int32_t* err;
};

// Partitions actually used: at least 2^min_log2 stages each, so a short batch
// is not spread thinner than a kernel's pipeline depth.
__device__ __forceinline__ int64_t eff_grid(int64_t S, int64_t launched, int min_log2) {
  const int64_t want = (S + (int64_t(1) << min_log2) - 1) >> min_log2;
  return want < 1 ? 1 : (want < launched ? want : launched);
}

__device__ __forceinline__ int seq_tokens(const Params& p, int b, int P) {
  if (p.kv_tokens) return max(0, p.kv_tokens[b]);
  return max(0, (p.kv_indptr[b + 1] - p.kv_indptr[b]) * P);
}

__device__ __forceinline__ int seq_mode(const Params& p, int b) {
  if (!p.mode_of_row) return CE_MODE_NONE;
  const int64_t row = p.rows ? p.rows[b] : b;
  return p.mode_of_row[row];
}

// Block-wide exclusive scan of one int64 per thread (sh: 32 words).
__device__ __forceinline__ int64_t block_excl_scan(int64_t v, int64_t* sh, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    int64_t run = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
      int64_t t = sh[w];
      sh[w] = run;
      run += t;
    }
    sh[31] = run;
  }
  __syncthreads();
  int64_t res = sh[warp] + x - v;
  total = sh[31];
  __syncthreads();
  return res;
}

__device__ __forceinline__ int cta_of_stage(int64_t x, int64_t S, int64_t grid) {
  return static_cast<int>(((x + 1) * grid - 1) / S);
}

}  // namespace decode

namespace host {

// Byte offsets of a decode call's workspace.  The partial records come last,
// so that the score data lies at the same place for every launch width.
struct DecodeLayout {
  size_t prefix, lse2, ul, tl, rec, total;
};
DecodeLayout decode_layout(int bs, int64_t cap, int H, int P, int flags, int grid);

}  // namespace host
}  // namespace ce
