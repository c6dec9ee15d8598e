// What the attention kernels over pages of codes share: the argument block and who takes which request.
#pragma once

#include "float8.cuh"

namespace attn8 {

// A request with at most this many (token, head-of-group) rows is a decode request: each is two of a product's 16 (or 32) columns.
__host__ __device__ inline int decode_rows(int g) { return g <= 8 ? 8 : g <= 16 ? 16 : 0; }

struct Params {
  const __nv_bfloat16* q;        // [T, Hq, HD]
  const float *k_scale, *v_scale;        // [pages, Hkv]
  __nv_bfloat16* out;            // [T, Hq * HD]
  const int32_t* block_table;    // [R, table_width]
  const int32_t* cu_q;           // [R + 1]
  const int32_t* kv_lens;        // [R]
  int table_width, R, Hq, Hkv, g, window, page;
  float scale_log2;              // scale * log2(e)
};

}  // namespace attn8
