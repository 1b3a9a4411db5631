// Arguments of the attention over the block-wise 8-bit KV cache, shared by its kernels.
#pragma once

#include "launchers.h"

namespace qw {

struct CachedPages {  // keys or values: [blocks, Hkv, block, D] codes, [blocks, Hkv] scales
  const uint8_t* codes;
  int64_t block_stride, head_stride, token_stride;
  const float* scale;
  int64_t scale_stride;
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
  int max_table_tokens;  // width * block: no request can see more
  float scale;
  float* part_o;    // partial outputs
  float* part_ml;   // their running maximum and sum
  int64_t* prefix;  // [B + 1]
};

int cached_attn_workers(int mt);
void cached_attention_rows(const CachedAttn& p, int D, int fmt, int mt, cudaStream_t stream);

}  // namespace qw
