// The parts of garuda_branches that its kernel files share: attention of drafted trees.
#pragma once

#include <atomic>

#include "common.cuh"

namespace branches {

// Numbers 0 .. N - 1 that a device is asked for once. Threads that are first together ask twice and get the same.
template <int N>
class AskedOnce {
  std::atomic<int> known_[gb::OncePerDevice::MAX_DEVICES][N] = {};       // one more than the number; 0: not asked for yet

 public:
  template <typename F>
  int get(int i, F ask) {
    const int d = gb::OncePerDevice::device();
    if (d < 0) return ask();
    int n = known_[d][i].load(std::memory_order_relaxed);
    if (n == 0) known_[d][i].store(n = ask() + 1, std::memory_order_relaxed);
    return n - 1;
  }
};

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

// What the attention's entry points are given, in one piece (a call of two dozen arguments takes its caller three microseconds longer). The caller
// packs the same fields in the same order, eight bytes each.
struct TreeCall {
  const void *q, *k_pool, *v_pool;
  void* out;
  const int32_t *block_table, *cu_q, *kv_lens, *positions, *mask;
  void *counters, *scratch, *stream;
  long long table_width, mask_words, T, R, pages, Hq, Hkv, head_dim, window, page_size, max_q_len, max_kv_len, dtype;
  double scale;
  TreeParams params() const {
    return {q, k_pool, v_pool, out, block_table, cu_q, kv_lens, positions, reinterpret_cast<const uint32_t*>(mask), pages, (int)table_width,
            (int)mask_words, (int)Hq, (int)Hkv, (int)(Hq / Hkv), (int)window, (int)page_size, (int)T, (int)R, (float)scale};
  }
};

}  // namespace branches
