// The parts of garuda_branches that its kernel files share: attention of drafted trees.
#pragma once

#include "common.cuh"

namespace branches {

// Attention of a request's drafted tokens over its pages. Token i of request r reads the keys of the context, positions 0 to
// kv_lens[r] - (cu_q[r + 1] - cu_q[r]) - 1 (with a window those above positions[i] - window), and those drafted tokens j of the request,
// which lie behind the context in the order of their numbers, for which bit j of its row of `mask` is set.
struct TreeParams {
  const void* q;                 // [T, Hq, hd]
  const void* k_pool;            // [pages, Hkv, page_size, hd]
  const void* v_pool;
  void* out;                     // [T, Hq * hd]
  const int32_t* block_table;    // [R, table_width]
  const int32_t* cu_q;           // [R + 1]
  const int32_t* kv_lens;        // [R]
  const int32_t* positions;      // [T]; read with a window only
  const uint32_t* mask;          // [T, mask_words]
  long long pages;
  int table_width, mask_words, Hq, Hkv, g, window, page_size, T, R;
  float scale;
};

}  // namespace branches
