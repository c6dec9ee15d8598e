// Bookkeeping of branches on the device: a drafted tree's positions and masks, the walk along its accepted tokens with the rows they
// left in the cache, and copies of pages and states for forked requests.
#include "branches.h"
#include "error_word.cuh"
#include "tc_common.cuh"

#include <climits>

GB_DEFINE_LAST_ERROR()

namespace {

using namespace tc;

// ------------------------------------------------------------------ tree layout
// parents[t]: the token of the same request, counted from its first, that token t continues; -1: the context. A chain of parents goes
// towards the front and ends at -1, else the token belongs to no branch: it stands at the context's end and reads nothing.
//   positions[t] = context + number of ancestors;   bit j of mask[t]: j is t or one of its ancestors
// and with a window fewer than `window` positions in front of it. A block a request, a thread a token: a walk along the parents in shared
// memory (30 clocks a step; a step's layers all read the result, so the walk's length matters once), then the bits from the
// highest word down, which the walk meets in that order.
constexpr int LAYOUT_THREADS = 128;
constexpr int LAYOUT_TOKENS = 8192;      // of one request (their parents are in shared memory)

__global__ void __launch_bounds__(LAYOUT_THREADS)
tree_layout_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ cu_q, const int32_t* __restrict__ kv_lens,
                   int32_t* __restrict__ positions, uint32_t* __restrict__ mask, const int words, const int window) {
  extern __shared__ int32_t up[];
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  const int r = blockIdx.x, first = cu_q[r], q_len = cu_q[r + 1] - first, ctx = kv_lens[r] - q_len;
  const int known = min(q_len, words * 32);          // (the mask has no bits for more)
  for (int i = threadIdx.x; i < known; i += LAYOUT_THREADS) up[i] = parents[first + i];
  __syncthreads();
  for (int i = threadIdx.x; i < q_len; i += LAYOUT_THREADS) {
    int depth = 0;
    bool rooted = i < known;
    for (int at = i; rooted;) {
      const int above = up[at];
      if (above == -1) break;
      rooted = above >= 0 && above < at;
      at = above, ++depth;
    }
    positions[first + i] = ctx + (rooted ? depth : 0);
    uint32_t* row = mask + (size_t)(first + i) * words;
    int next = words - 1;                            // the highest word that is not written yet
    if (rooted) {
      uint32_t bits = 0;
      int word = i >> 5;
      for (int at = i, back = 0; at >= 0 && (window <= 0 || back < window); at = up[at], ++back) {
        if ((at >> 5) != word) {
          for (; next > word; --next) row[next] = 0;
          row[next--] = bits;
          word = at >> 5, bits = 0;
        }
        bits |= 1u << (at & 31);
      }
      for (; next > word; --next) row[next] = 0;
      row[next--] = bits;
    }
    for (; next >= 0; --next) row[next] = 0;
  }
}

// ------------------------------------------------------------------ acceptance
// From a request's first token on: of the tokens that continue token a (parents[c] = a) the first one that is what the model chose
// behind a (tokens[c] = targets[a]) is accepted, and so on until there is none. path[r] = the accepted tokens, the first among them,
// then -1; kept[r]: how many; next_tokens[r] = targets of the last. Row ctx + path[i] of every array's pages goes to row ctx + i.
//
// Every block of a request makes the same walk (a few microseconds' worth of waiting at most, and no block waits for another), then moves its
// share of the rows. A thread has its vectors of every row to itself and path is ascending, path[i] >= i: read in that order, some rows at a time before
// any of them is written, no row is overwritten before it has been read. (Four: 64 requests of 64 tokens, 43 MB of rows read and written, take 13.0 us; eight, for
// which registers leave fewer blocks on an SM, 15.9, two 13.4.) Bound by the way to the rows (lengths, then the tree and its pages, then the rows: 3 us for
// one small tree) and by their pieces of 256 bytes, which lie apart: 3.3 TB/s.
constexpr int ACCEPT_THREADS = 256;
constexpr int ACCEPT_TOKENS = 8192;
constexpr int AHEAD = 4;

struct Arrays {
  static constexpr int MOST = 64;
  uint8_t* at[MOST];          // [calls, pages, heads, page_size, row] each
  int heads[MOST], row_bytes[MOST];
  int first[MOST + 1];        // calls of the arrays in front
  int n;
};

template <typename V>
__global__ void __launch_bounds__(ACCEPT_THREADS)
tree_accept_kernel(const int32_t* __restrict__ tokens, const int32_t* __restrict__ targets, const int32_t* __restrict__ parents,
                   const int32_t* __restrict__ cu_q, const int32_t* __restrict__ kv_lens, int32_t* __restrict__ path, const int path_width,
                   int32_t* __restrict__ kept, int32_t* __restrict__ next_tokens, const __grid_constant__ Arrays arrays, const long long pages,
                   const int32_t* __restrict__ block_table, const int table_width, const int page_size, const int most, const int per_block) {
  extern __shared__ int2 smem[];
  int2* const from = smem;                      // [most]: page and line of the rows (page -1: no move)
  int2* const to = from + most;
  int32_t* const walk = reinterpret_cast<int32_t*>(to + most);          // [most]
  int32_t* const pages_s = walk + most;         // [most + 1]: from the context's end on
  int32_t* const follow = reinterpret_cast<int32_t*>(from);             // [most]: the token accepted behind each (until the rows are known)
  int32_t* const wanted = reinterpret_cast<int32_t*>(to);               // [most]: targets (likewise)
  __shared__ int kept_s, moved_s;
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  const int r = blockIdx.y, first = cu_q[r], q_len = min(cu_q[r + 1] - first, most), ctx = kv_lens[r] - (cu_q[r + 1] - first);
  const bool moves = arrays.n > 0 && ctx >= 0;
  const int first_entry = moves ? ctx / page_size : 0, last_entry = moves ? min(table_width, (ctx + q_len - 1) / page_size + 1) : 0;
  for (int i = threadIdx.x; i < q_len; i += ACCEPT_THREADS) follow[i] = INT_MAX, wanted[i] = targets[first + i];
  for (int i = first_entry + threadIdx.x; i < last_entry; i += ACCEPT_THREADS) pages_s[i - first_entry] = block_table[(size_t)r * table_width + i];
  for (int i0 = 0; i0 < q_len; i0 += ACCEPT_THREADS) {
    const int i = i0 + threadIdx.x, above = i < q_len ? parents[first + i] : -1, token = i < q_len ? tokens[first + i] : 0;
    if (i0 == 0) __syncthreads();               // (behind the loads, which are on their way together)
    if (above >= 0 && above < i && token == wanted[above]) atomicMin(&follow[above], i);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0, in_place = 0;                    // (the first tokens of a path may be where they belong, none behind one that is not)
    for (int at = 0; at < q_len; at = follow[at]) in_place += at == n, walk[n++] = at;
    kept_s = n, moved_s = in_place;
  }
  __syncthreads();
  const int n = kept_s, moved = moved_s;
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < path_width; i += ACCEPT_THREADS) path[(size_t)r * path_width + i] = i < n ? walk[i] : -1;
    if (threadIdx.x == 0) kept[r] = n, next_tokens[r] = n > 0 ? targets[first + walk[n - 1]] : -1;
  }
  if (!moves || moved == n) return;
  for (int i = moved + threadIdx.x; i < n; i += ACCEPT_THREADS) {
    auto line = [&](int slot) {
      const int entry = slot / page_size, page = entry < last_entry ? pages_s[entry - first_entry] : -1;
      return make_int2(page < pages ? page : -1, slot % page_size);
    };
    const int2 a = line(ctx + walk[i]), b = line(ctx + i);
    from[i] = make_int2(b.x >= 0 ? a.x : -1, a.y), to[i] = b;
  }
  __syncthreads();
  // this block's calls, of all arrays in a row; its threads have (call, head, vector) places
  const int begin = blockIdx.x * per_block, end = min(arrays.first[arrays.n], begin + per_block);
  int k = 0;
  for (int call = begin; call < end;) {
    while (arrays.first[k + 1] <= call) ++k;
    const int vectors = arrays.row_bytes[k] / (int)sizeof(V), per_call = arrays.heads[k] * vectors;
    const int calls = min(end, arrays.first[k + 1]) - call;
    const size_t line_bytes = arrays.row_bytes[k], head_bytes = line_bytes * page_size, page_bytes = head_bytes * arrays.heads[k];
    for (int x = threadIdx.x; x < calls * per_call; x += ACCEPT_THREADS) {
      const int head = x % per_call / vectors, vector = x % vectors;
      uint8_t* const base = arrays.at[k] + (size_t)(call - arrays.first[k] + x / per_call) * pages * page_bytes + head * head_bytes +
                            vector * sizeof(V);
      auto place = [&](int2 where) { return reinterpret_cast<V*>(base + where.x * page_bytes + where.y * line_bytes); };
      for (int i0 = moved; i0 < n; i0 += AHEAD) {
        V v[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e)
          if (i0 + e < n && from[i0 + e].x >= 0) v[e] = *place(from[i0 + e]);
#pragma unroll
        for (int e = 0; e < AHEAD; ++e)
          if (i0 + e < n && from[i0 + e].x >= 0) *place(to[i0 + e]) = v[e];
      }
    }
    call += calls;
  }
}

// ------------------------------------------------------------------ copies of entries
// arrays [outer, entries, bytes]: entry source[i] goes to entry target[i], in every outer row, for all i, as if all were read before any is
// written. A source or target outside the array is no copy; of several to one target the last counts.
//
// Bound by the memory's rate. A piece of work is a column of the array: some bytes of every entry, which the block brings to shared memory
// for all copies (a bulk copy each), and once all are there sends back. So whatever is overwritten has been read, by the same
// block, and blocks have nothing to do with one another. Columns that do not start on 16 bytes are copied by the threads.
constexpr int COPY_THREADS = 128;
constexpr int MOST_COPIES = 1024;

struct CopyArrays {
  static constexpr int MOST = 96;
  uint8_t* at[MOST];
  long long bytes[MOST];          // of an entry
  int outer[MOST], entries[MOST];
  int n;
};

struct CopyShared {
  uint64_t full;
  int n;
  int source[MOST_COPIES], target[MOST_COPIES], listed[MOST_COPIES];
};

template <typename U>             // what the threads copy, where they do (U = uint4: bulk copies)
__global__ void __launch_bounds__(COPY_THREADS)
copy_entries_kernel(const __grid_constant__ CopyArrays arrays, const int32_t* __restrict__ source, const int32_t* __restrict__ target,
                    const int copies, const int column) {
  constexpr bool BULK = sizeof(U) == 16;
  extern __shared__ __align__(128) uint8_t columns[];
  __shared__ CopyShared sh;
  const uint32_t bar = smem_u32(&sh.full), base = smem_u32(columns);
  if (BULK && threadIdx.x == 0) {
    mbar_init(bar, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  for (int i = threadIdx.x; i < copies; i += COPY_THREADS) sh.listed[i] = target[i];
  __syncthreads();
  uint32_t phase = 0;
  bool ok = true;
  int valid_for = -1;               // the entries that the list has been made for
  int n = 0;
  long long work = blockIdx.x;      // pieces: array by array, outer row by outer row
  for (int k = 0; k < arrays.n && ok; ++k) {
    const long long bytes = arrays.bytes[k], per_row = (bytes + column - 1) / column, pieces = per_row * arrays.outer[k];
    if (work < pieces && valid_for != arrays.entries[k]) {
      // the copies that count, for arrays of so many entries
      valid_for = arrays.entries[k];
      __syncthreads();
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < copies; i += COPY_THREADS) {
        const int a = source[i], b = sh.listed[i];
        bool counts = a >= 0 && a < valid_for && b >= 0 && b < valid_for;
        // (a later copy to the same target that is none does not count against this one)
        for (int j = i + 1; counts && j < copies; ++j)
          if (sh.listed[j] == b && (unsigned)source[j] < (unsigned)valid_for) counts = false;
        if (counts && a != b) {
          const int at = atomicAdd(&sh.n, 1);
          sh.source[at] = a, sh.target[at] = b;
        }
      }
      __syncthreads();
      n = sh.n;
    }
    for (; work < pieces && ok; work += gridDim.x) {
      const long long off = work % per_row * column;
      const uint32_t size = (uint32_t)min((long long)column, bytes - off);
      uint8_t* const row = arrays.at[k] + (work / per_row) * arrays.entries[k] * bytes + off;
      if (n == 0) continue;
      if (BULK) {
        if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, size * n);
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += COPY_THREADS)
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(base + i * column),
                       "l"(row + sh.source[i] * bytes), "r"(size), "r"(bar) : "memory");
        const bool came = mbar_wait(bar, phase);
        phase ^= 1;
        if (!came) gb_err::report(ERR_WAIT_FULL);
        ok = __syncthreads_and(came);
        if (!ok) {                    // what is still in flight needs microseconds to land
          const unsigned long long t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 2000000ull) {}
          break;
        }
        for (int i = threadIdx.x; i < n; i += COPY_THREADS)
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(row + sh.target[i] * bytes), "r"(base + i * column),
                       "r"(size) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncthreads();
      } else {
        const int units = size / (int)sizeof(U);
        for (int x = threadIdx.x; x < n * units; x += COPY_THREADS)
          *reinterpret_cast<U*>(columns + (x / units) * column + (x % units) * sizeof(U)) =
              *reinterpret_cast<const U*>(row + sh.source[x / units] * bytes + (x % units) * sizeof(U));
        __syncthreads();
        for (int x = threadIdx.x; x < n * units; x += COPY_THREADS)
          *reinterpret_cast<U*>(row + sh.target[x / units] * bytes + (x % units) * sizeof(U)) =
              *reinterpret_cast<const U*>(columns + (x / units) * column + (x % units) * sizeof(U));
        __syncthreads();
      }
    }
    work -= pieces;                 // (the place in the next array's pieces: all arrays' are one row)
  }
}

}  // namespace

GB_EXPORT int gb_tree_layout(const int32_t* parents, const int32_t* cu_q, const int32_t* kv_lens, int32_t* positions, int32_t* mask, int words,
                             int window, int R, int max_q_len, void* stream) {
  if (max_q_len > LAYOUT_TOKENS) return gb::fail(GB_UNSUPPORTED, "tree_layout: %d drafted tokens of one request (at most %d)", max_q_len, LAYOUT_TOKENS);
  if (R <= 0) return GB_OK;
  return gb::check_pdl_launch(gb::launch_pdl(tree_layout_kernel, dim3(R), dim3(LAYOUT_THREADS), sizeof(int32_t) * 32 * words, (cudaStream_t)stream,
                                             dim3(1), parents, cu_q, kv_lens, positions, reinterpret_cast<uint32_t*>(mask), words, window),
                              "tree_layout");
}

// What the caller packs, eight bytes each (see TreeCall).
struct AcceptCall {
  const int32_t *tokens, *targets, *parents, *cu_q, *kv_lens;
  int32_t *path, *kept, *next_tokens;
  const int32_t* block_table;
  const long long* pools;          // n times {address, calls, heads, bytes of a row}: arrays [calls, pages, heads, page_size, row bytes]
  void* stream;
  long long n, pages, path_width, table_width, page_size, R, max_q_len;
};
GB_EXPORT int gb_tree_accept(const AcceptCall* call) {
  const int n = (int)call->n, R = (int)call->R, max_q_len = (int)call->max_q_len;
  if (n > Arrays::MOST) return gb::fail(GB_UNSUPPORTED, "tree_accept: %d pools (at most %d)", n, Arrays::MOST);
  if (max_q_len > ACCEPT_TOKENS) return gb::fail(GB_UNSUPPORTED, "tree_accept: %d drafted tokens of one request (at most %d)", max_q_len, ACCEPT_TOKENS);
  if (R <= 0) return GB_OK;
  Arrays a{};
  a.n = n;
  uintptr_t all = 0;
  for (int k = 0; k < n; ++k) {
    const long long* pool = call->pools + 4 * k;
    a.at[k] = (uint8_t*)pool[0], a.heads[k] = (int)pool[2], a.row_bytes[k] = (int)pool[3];
    a.first[k + 1] = a.first[k] + (int)pool[1];
    all |= (uintptr_t)pool[0] | (uintptr_t)pool[3];
  }
  const int rows = a.first[n];
  // a few more blocks than run at once (six of 256 threads an SM; exactly as many 13.8 us, twice as many 17): each walks its request's tree
  const int room = 8 * gb::sm_count();
  const int per_block = rows > 0 ? (int)(((long long)rows * R + room - 1) / room) : 1, blocks = rows > 0 ? (rows + per_block - 1) / per_block : 1;
  const size_t smem = 24 * (size_t)max_q_len + 4;
  auto launch = [&](auto vector) {
    const auto kernel = tree_accept_kernel<decltype(vector)>;
    static gb::OncePerDevice configured;          // (one per type)
    if (configured.needed()) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 24 * ACCEPT_TOKENS + 4);
      if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "tree_accept: %s", cudaGetErrorString(e));
      configured.done();
    }
    return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3(blocks, R), dim3(ACCEPT_THREADS), smem, (cudaStream_t)call->stream, dim3(1), call->tokens,
                                               call->targets, call->parents, call->cu_q, call->kv_lens, call->path, (int)call->path_width, call->kept,
                                               call->next_tokens, a, call->pages, call->block_table, (int)call->table_width, (int)call->page_size, max_q_len,
                                               per_block), "tree_accept");
  };
  if (all % 16 == 0) return launch(uint4{});
  if (all % 4 == 0) return launch(uint32_t{});
  return launch(uint16_t{});
}

struct CopyCall {
  const int32_t *source, *target;
  const long long* arrays;         // n times {address, outer, entries, bytes}
  void* stream;
  long long n, copies;
};
GB_EXPORT int gb_copy_entries(const CopyCall* call) {
  const int n = (int)call->n, copies = (int)call->copies;
  if (copies > MOST_COPIES) return gb::fail(GB_UNSUPPORTED, "copy_entries: %d copies (at most %d)", copies, MOST_COPIES);
  if (copies <= 0) return GB_OK;
  // Shared memory for one column of every copy: a quarter of an SM's, as long as that gives columns of 512 bytes, else more.
  for (int k0 = 0; k0 < n; k0 += CopyArrays::MOST) {
    CopyArrays a{};
    uintptr_t all = 0;
    long long widest = 0;
    for (int k = k0; k < n && a.n < CopyArrays::MOST; ++k, ++a.n) {
      const long long* array = call->arrays + 4 * k;
      a.at[a.n] = (uint8_t*)array[0], a.outer[a.n] = (int)array[1], a.entries[a.n] = (int)array[2], a.bytes[a.n] = array[3];
      all |= (uintptr_t)array[0] | (uintptr_t)array[3];
      widest = widest > array[3] ? widest : array[3];
    }
    constexpr int QUARTER = 40 * 1024, WHOLE = 200 * 1024;
    long long column = QUARTER / copies >= 512 ? QUARTER / copies : WHOLE / copies < 512 ? WHOLE / copies : 512;
    column = column >= 128 ? column / 128 * 128 : column / 16 * 16;
    if (column > widest) column = (widest + 15) / 16 * 16;
    long long pieces = 0;
    for (int k = 0; k < a.n; ++k) pieces += (a.bytes[k] + column - 1) / column * a.outer[k];
    if (pieces == 0) continue;
    const int smem = (int)(column * copies);
    const int beside = 224 * 1024 / (smem + (int)sizeof(CopyShared) + 1024);          // blocks that fit an SM
    const long long room = (long long)gb::sm_count() * (beside > 4 ? 4 : beside);
    auto launch = [&](auto unit) {
      const auto kernel = copy_entries_kernel<decltype(unit)>;
      static gb::OncePerDevice configured;
      if (configured.needed()) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, WHOLE);
        if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "copy_entries: %s", cudaGetErrorString(e));
        configured.done();
      }
      return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3((unsigned)(pieces < room ? pieces : room)), dim3(COPY_THREADS), smem, (cudaStream_t)call->stream,
                                                 dim3(1), a, call->source, call->target, copies, (int)column), "copy_entries");
    };
    const int rc = all % 16 == 0 ? launch(uint4{}) : all % 4 == 0 ? launch(uint32_t{}) : launch(uint8_t{});
    if (rc) return rc;
  }
  return GB_OK;
}

GB_EXPORT int gb_branches_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_branches_set_error_sink(int* host_word) { return gb_err::set_sink(host_word); }
