// Arguments of the attention over the block-wise 8-bit KV cache, shared by its kernels.
#pragma once

#include "divisor.cuh"
#include "launchers.h"

namespace qw {

// Keys or values: [blocks, Hkv, block, D] codes, [blocks, Hkv] scales. Strides below 2^32 (checked where tensors come in),
// so that an address takes 32 x 32-bit products.
struct CachedPages {
  const uint8_t* codes;
  uint32_t block_stride, head_stride, token_stride;
  const float* scale;
  uint32_t scale_stride;
};

struct CachedAttn {
  const bf16* q;  // [T, Hkv * group, D]
  int64_t q_token, q_head;
  bf16* out;
  int64_t o_token, o_head;
  CachedPages k, v;
  const int* table;  // [B, width]
  int64_t table_stride;
  const int* context;      // [B]
  const int* query_start;  // [B + 1]
  int T, B, Hkv, group, block, blocks;
  Divisor by_group, by_block;
  int max_table_tokens;  // width * block: no request can see more
  float scale;
  float* part_o;    // partial outputs
  float* part_ml;   // their running maximum and sum
  int64_t* prefix;  // [B + 1]
};

// A query row enters f16 divided by a power of two that brings its largest number to [2^14, 2^15): bf16 numbers down to 2^-31 of
// it are then exact in f16 (8 bits, multiples of 2^-24), and smaller ones are off by at most 2^-39 of it, far below the
// rounding of the 32-bit sums. (Brought to [1, 2), numbers below 2^-17 of the largest lost bits, which counted where
// large keys met them.) A sum of 128 products with codes stays below 2^15 * 448 * 128 < 2^31.
constexpr int kQueryTop = 14;

// The rows of q that belong to request b; offsets outside [0, T] are cut, so that no row outside q is touched.
struct NewRows {
  int first, n;
};
__device__ __forceinline__ NewRows new_rows(const CachedAttn& p, int b) {
  const int first = min(max(p.query_start[b], 0), p.T);
  return {first, min(max(p.query_start[b + 1], 0), p.T) - first};
}

// The request that row `tok` of q belongs to (the last one that begins at or before it), for a whole warp: the offsets are
// read side by side, not one after another as in a binary search.
__device__ __forceinline__ int request_of(const CachedAttn& p, int tok) {
  const int lane = threadIdx.x % 32;
  int n = 0;
  for (int b0 = 0; b0 < p.B; b0 += 128) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + i * 32 + lane;
      n += __popc(__ballot_sync(0xffffffffu, b < p.B && p.query_start[b < p.B ? b : 0] <= tok));
    }
  }
  return max(n - 1, 0);
}

// tcgen05 kernel for prompts (head_dim 64 and 128), `splits` parts of the keys; rows and resident blocks of threads per SM
constexpr int prompt_rows(int D) { return D == 64 ? 128 : 256; }
constexpr int prompt_per_sm(int D) { return D == 64 ? 2 : 1; }
void cached_attention_prompt(const CachedAttn& p, int D, int fmt, int tiles_max, int splits, cudaStream_t stream);

}  // namespace qw
