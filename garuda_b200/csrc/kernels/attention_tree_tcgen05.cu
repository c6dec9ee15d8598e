// Attention of drafted trees over the paged cache on the fifth-generation tensor cores.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j   over the context's keys and those drafted tokens j whose bit is set in i's mask
// (garuda/src/llama/mod.rs:793-818 with another set of keys; the window garuda/src/cache/mod.rs:333-338; query head h reads key/value
// head h / g).
//
// What bounds it: a request's context is read once per key/value head for a few to a few hundred query rows, (token, head-of-group)
// pairs. At 128 rows a byte of the cache is worth 128 operations, at 256 rows the products take as long as the bytes. So both products
// of a tile are tcgen05.mma with 128 rows, few as the rows may be: at 128 keys and heads of 128 they take 1,100 clocks for 64 KB, which
// one SM's share of the memory's rate needs 2,700 for.
//
// The work is the row of all tiles of 128 keys, of all requests, heads and blocks of 128 rows, cut into stretches of equal cost, one for
// every CTA (a CTA an SM), whatever the requests' lengths are. A stretch may begin and end inside a block's keys: its pieces' sums go to
// scratch memory, with their maxima and denominators, and the CTA that counts the last of a block's pieces joins them in the order of the keys,
// so that the result does not depend on who comes last. Few blocks of few tiles are a thread-block cluster's each, which joins in shared memory.
//   warp 0     the pieces of the stretch; queries (a box [tokens][group][64]) and keys by TMA, a box per page and 64 channels. What lies outside the
//              pool (no page: -1) reads as zeros
//   warp 10    values, in a ring of their own (keys are needed two tiles before: in one warp they waited behind the values)
//   warp 1     one elected lane issues the products: S = Q K^T two tiles ahead, O += P V (P from tensor memory)
//   warps 2-9  two groups of 128 threads; a thread has a row and 64 keys of every tile: an attention stream of its own, whose reference
//              maximum follows the running one when that has grown by 2^8. Warps whose rows are all behind the last only keep count
// A tile takes 2,900 to 3,000 clocks of a stretch, what its bytes take at the memory's rate: 2,000 are a warp's softmax (of which 1,024 the exponentials, sixteen a
// clock and SM), 1,100 the products, which run beside the other tile's. 32 requests of 4,096 keys, 24 tokens: 104 us, of which the bytes are 84; lengths from
// 256 to 8,191: 106 (equal numbers of tiles: 153). Call behind call the power limit takes the clock from 1,965 to 1,690 MHz, and the latter 117:
// fewer instructions are a higher clock (scores and sums one by one, not two at a time: 120.5; a quarter of the
// exponentials as polynomials on the other pipes: 133; the groups on alternate tiles instead of halves, each with a row's 128 keys in two walks: 109 and 122.5).
// Tiles that hold a key which some row does not read are masked by 64 bits a thread, made of the row's bits and limits. Their values
// are looked at: a row of values that no query may read is cleared (it holds whatever was there), and one with an infinity or NaN
// is cleared too and told to the rows, of which those that read it become NaN and the others are left alone (0 * inf would
// spoil them). Every wait is bounded.
#include <cuda_bf16.h>

#include "branches.h"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace {

using namespace tc;
using branches::TreeParams;

constexpr int QROWS = 128;          // query rows of a block
constexpr int KT = 128;             // keys of a tile
constexpr int GROUPS = 2;           // softmax groups: each walks its own half of every key tile
constexpr int GK = KT / GROUPS;
constexpr int ROW_BYTES = 128;      // one swizzled row: 64 channels
constexpr int BLOCK_BYTES = 128 * ROW_BYTES;
constexpr int THREADS = 96 + GROUPS * 128;           // warps: keys, products, softmax (eight), values
constexpr int TMEM_COLS = 512;
constexpr int S_BUFS = 2;           // S buffers: the S products run this many tiles ahead
constexpr int O_COL0 = S_BUFS * KT;
constexpr float RESCALE_ABOVE = 8.f;                // in powers of two
constexpr int MIN_STRETCH = 4;                      // of shorter ones the joining takes longer than the tiles
constexpr int BLOCK_COST = 4;                       // what a block of rows costs beside its tiles, in tiles (two: 113 us for 110, 130 for 123 at the lower clock)
constexpr int MAX_REQUESTS = 2048;                  // of one launch (their places are in shared memory)
constexpr int COUNTERS = 1024;                      // one per CTA, and so no more CTAs

template <int HD>
struct Shape {
  static constexpr int BLOCKS = HD / 64;            // blocks of 64 channels: one swizzled 128-byte row each
  static constexpr int BYTES = BLOCKS * BLOCK_BYTES;                  // of 128 rows of queries, keys or values
  static constexpr int K_STAGES = HD == 64 ? 4 : 2, V_STAGES = HD == 64 ? 5 : 3;
  static constexpr int TILE_BYTES = (1 + K_STAGES + V_STAGES) * BYTES;
  // a stage of keys is given back by the tensor core where stages are few, else by a softmax thread that has seen the scores
  // (a commit costs the issuing thread as much as two products)
  static constexpr bool KEYS_FREED_BY_COMMIT = K_STAGES < S_BUFS + 1;
  static constexpr int CH = HD / GROUPS;            // channels that a group writes out
  static constexpr int PART_FLOATS = QROWS * (HD + 2);                // a piece's sums, maxima and denominators
  static_assert(GK == 64 && O_COL0 + GROUPS * HD <= TMEM_COLS, "tensor memory layout");
};

// A piece: tiles first .. first + count (0: there is none) of the n of one request's block of rows and head. The row of all blocks' costs,
// a tile each and BLOCK_COST for a block, is what is cut into stretches.
struct Piece {
  int r, kvh, tok0, nrows, q_begin, ctx, kv_len;      // of the request: its first token, its context and all its keys
  int lo, tile0, first, n, count;                     // first key that any row reads; the tile that it lies in
  int at, next;                                       // in the row of costs: the block's place, and what comes behind the piece
};

struct Misc {
  uint64_t q_full, q_empty, met, k_full[4], k_empty[4], v_full[5], v_empty[5];
  uint64_t s_ready[S_BUFS], p_ready[S_BUFS], o_ready[2], looked[GROUPS];
  uint32_t tmem_base;
  int abort, last, total, scan[THREADS / 32];
  Piece piece[2], own;                    // two pieces in turn, from the warp of the keys; CLUSTER: the CTA's
  uint32_t bad[2][GROUPS][2];             // keys of a masked tile whose values are not finite, a bit each, two such tiles in turn
  float2 ml[2][GROUPS][QROWS];            // the groups' reference maxima and denominators, two pieces in turn
};

__device__ __forceinline__ float fast_exp2(float x) {      // about 2^-22 relative; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
typedef unsigned long long Two;            // two floats, for one instruction
__device__ __forceinline__ Two two(float a, float b) {
  Two d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 apart(Two a) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
  return d;
}
__device__ __forceinline__ Two fma_two(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Two add_two(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void clear_shared_v4(uint32_t addr) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0u) : "memory");
}
// whether one of two bfloat16 is an infinity or NaN
__device__ __forceinline__ bool not_finite(uint32_t w) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; }

// Four bytes to sixteen of another CTA's shared memory (an address of the cluster's window).
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// A row's result of several pieces: their sums with weights 2^(m - the largest m), over the denominators' sum. m is in powers of two.
template <int FOURS>               // of channels
struct Join {
  float m = -INFINITY, l = 0.f;
  float4 t[FOURS] = {};
  __device__ __forceinline__ void add(float2 ml, const float4 (&v)[FOURS]) {
    if (ml.x == -INFINITY && ml.y == 0.f) return;               // no key of this piece
    const float top = fmaxf(m, ml.x);
    // (without a reference there is nothing yet, or what is no number)
    const float keep = m == -INFINITY ? (l == 0.f ? 0.f : NAN) : fast_exp2(m - top), more = ml.x == -INFINITY ? NAN : fast_exp2(ml.x - top);
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
      t[i].x = t[i].x * keep + v[i].x * more, t[i].y = t[i].y * keep + v[i].y * more;
      t[i].z = t[i].z * keep + v[i].z * more, t[i].w = t[i].w * keep + v[i].w * more;
    }
    l = l * keep + ml.y * more, m = top;
  }
  __device__ __forceinline__ void store(__nv_bfloat16* to) const {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < FOURS; i += 2)
      *reinterpret_cast<uint4*>(to + 4 * i) = make_uint4(pack_bf16(t[i].x * inv, t[i].y * inv), pack_bf16(t[i].z * inv, t[i].w * inv),
                                                         pack_bf16(t[i + 1].x * inv, t[i + 1].y * inv), pack_bf16(t[i + 1].z * inv, t[i + 1].w * inv));
  }
};

// Joins a block's pieces, of the CTAs c0 to c1, in this order: by the 256 threads of the softmax warps. (A function of its own: its registers are
// not the tiles' loop's.) A thread has a row and a share of the channels, so many fours of so many pieces at a time: that many loads are on their way.
template <int HD, int AT_ONCE, int FOURS>
__device__ __forceinline__ void join_by(const float* __restrict__ parts, int c0, int c1, int nrows, __nv_bfloat16* __restrict__ out, int g, int Hq) {
  const int x = threadIdx.x - 64, rows = (nrows + 31) & ~31, shares = GROUPS * 128 / rows, row = x % rows, share = x / rows;
  const int mine = HD / 4 / shares;                              // fours of channels
  if (share >= shares || row >= nrows) return;
  auto part_of = [&](int cta) { return parts + ((size_t)cta * 2 + (cta == c0 ? 1 : 0)) * Shape<HD>::PART_FLOATS; };
  __nv_bfloat16* const to = out + ((size_t)(row / g) * Hq + row % g) * HD;
#pragma unroll 1
  for (int f0 = share * mine; f0 < (share + 1) * mine; f0 += FOURS) {
    Join<FOURS> join;
#pragma unroll 1
    for (int cta = c0; cta <= c1; cta += AT_ONCE) {
      float2 ml[AT_ONCE];
      float4 v[AT_ONCE][FOURS];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const float* from = part_of(min(cta + u, c1));
        ml[u] = __ldcg(reinterpret_cast<const float2*>(from + QROWS * HD + row * 2));
#pragma unroll
        for (int i = 0; i < FOURS; ++i) v[u][i] = __ldcg(reinterpret_cast<const float4*>(from) + (f0 + i) * QROWS + row);
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
        if (cta + u <= c1) join.add(ml[u], v[u]);
    }
    join.store(to + f0 * 4);
  }
}
template <int HD>
__device__ __noinline__ void join_pieces(const float* __restrict__ parts, int c0, int c1, int nrows, __nv_bfloat16* __restrict__ out, int g, int Hq) {
  // (more loads at once: the whole kernel runs short of registers)
  if (c1 - c0 == 1 && nrows > 32) join_by<HD, 2, 4>(parts, c0, c1, nrows, out, g, Hq);          // (up to 32 rows: a thread has two or four fours)
  else join_by<HD, 4, 2>(parts, c0, c1, nrows, out, g, Hq);
}

// CLUSTER: a block of rows and a head is a thread-block cluster's, of `ranks` CTAs, which share its keys; else CTAs have stretches.
template <int HD, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 1)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map, const TreeParams p, const int box_tokens, const int min_stretch,
                         const int ranks, const int most_blocks, float* __restrict__ parts, int* __restrict__ counters) {
  using S = Shape<HD>;
  constexpr int BLOCKS = S::BLOCKS, K_STAGES = S::K_STAGES, V_STAGES = S::V_STAGES, CH = S::CH;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Misc& mc = *reinterpret_cast<Misc*>(smem_raw + S::TILE_BYTES);
  int* const cost = reinterpret_cast<int*>(smem_raw + S::TILE_BYTES + sizeof(Misc));     // [R + 1]: of the requests in front
  int* const begin_s = cost + p.R + 1;                                                   // [R + 1]: cu_q
  int* const len_s = begin_s + p.R + 1;                                                  // [R]: kv_lens

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t q_s = smem_u32(smem_raw), k_s = q_s + S::BYTES, v_s = k_s + K_STAGES * S::BYTES;
  if ((q_s & 1023u) != 0) {                                        // the swizzle needs it; never seen
    if (threadIdx.x == 0) gb_err::report(ERR_WAIT_DRAIN);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&mc.q_full), 1);
    mbar_init(smem_u32(&mc.q_empty), GROUPS * 4 + 1);
    mbar_init(smem_u32(&mc.met), GROUPS * 4);
    for (int b = 0; b < S_BUFS; ++b) {
      mbar_init(smem_u32(&mc.s_ready[b]), 1);
      mbar_init(smem_u32(&mc.p_ready[b]), GROUPS * 128);
    }
    for (int s = 0; s < K_STAGES; ++s) mbar_init(smem_u32(&mc.k_full[s]), 1), mbar_init(smem_u32(&mc.k_empty[s]), 1);
    for (int s = 0; s < V_STAGES; ++s) mbar_init(smem_u32(&mc.v_full[s]), 1), mbar_init(smem_u32(&mc.v_empty[s]), 1);
    mbar_init(smem_u32(&mc.o_ready[0]), 1);
    mbar_init(smem_u32(&mc.o_ready[1]), 1);
    for (int g = 0; g < GROUPS; ++g) mbar_init(smem_u32(&mc.looked[g]), 4);
    mc.abort = 0, mc.total = 0;
    fence_barrier_init();
    fence_proxy_async();
    prefetch_tensormap(&q_map);
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&mc.tmem_base), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = mc.tmem_base;
  volatile int* abort_s = &mc.abort;
  gb::pdl_launch_dependents();
  gb::pdl_wait();      // everything, the lengths among it, may come from the kernels in front

  // ---- the tiles of every request
  const int tokens_per_block = QROWS / p.g;
  auto low_of = [&](int ctx) { return p.window > 0 ? max(0, ctx + 1 - p.window) : 0; };
  auto tiles_of = [&](int q_len, int kv_len) {       // of one head and block of rows: one at least, without keys too
    if (q_len <= 0) return 0;
    return (max(1, kv_len) - 1) / KT + 1 - low_of(max(0, kv_len - q_len)) / KT;
  };
  for (int r0 = 0; !CLUSTER && r0 < p.R; r0 += THREADS) {
    const int r = r0 + threadIdx.x;
    int n = 0;
    if (r < p.R) {
      const int q0 = p.cu_q[r], q1 = p.cu_q[r + 1], kv = p.kv_lens[r];
      begin_s[r] = q0, len_s[r] = kv;
      if (r + 1 == p.R) begin_s[r + 1] = q1;
      n = tiles_of(q1 - q0, kv);
      if (n > 0) n = (n + BLOCK_COST) * ((q1 - q0 + tokens_per_block - 1) / tokens_per_block) * p.Hkv;
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) mc.scan[warp] = inc;
    __syncthreads();
    int before = mc.total;
    for (int w = 0; w < warp; ++w) before += mc.scan[w];
    before += inc;
    if (r < p.R) {
      cost[r] = before - n;
      if (r + 1 == p.R) cost[r + 1] = before;
    }
    __syncthreads();
    if (threadIdx.x == THREADS - 1) mc.total = before;
    __syncthreads();
  }
  const int total = CLUSTER ? 0 : cost[p.R];
  const int stretch = max(min_stretch, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const int a_begin = (int)min((long long)total, (long long)blockIdx.x * stretch), a_end = min(total, a_begin + stretch);

  auto piece_at = [&](int a) {             // the piece that begins there or behind; count 0: the stretch has no more
    Piece w;
    w.count = 0;
    while (a < a_end) {
      int lo = 0, hi = p.R;                // the last request that begins at or before `a` (of several at the same place it has tiles)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cost[mid] <= a) lo = mid;
        else hi = mid;
      }
      w.r = lo, w.q_begin = begin_s[lo], w.kv_len = len_s[lo];
      const int q_len = begin_s[lo + 1] - w.q_begin, blocks = (q_len + tokens_per_block - 1) / tokens_per_block;
      w.ctx = max(0, w.kv_len - q_len);
      w.lo = low_of(w.ctx), w.tile0 = w.lo / KT;
      w.n = tiles_of(q_len, w.kv_len);
      const int per = w.n + BLOCK_COST, rem = a - cost[lo], unit = rem / per;
      w.first = rem - unit * per;
      w.at = a - w.first;
      if (w.first >= w.n) {                // what the block costs beside its tiles
        a = w.at + per;
        continue;
      }
      w.kvh = unit / blocks;               // (a head's blocks of rows one behind the other: they read the same keys)
      w.tok0 = unit % blocks * tokens_per_block;
      w.nrows = min(tokens_per_block, q_len - w.tok0) * p.g;
      w.count = min(w.n - w.first, a_end - a);
      w.next = a + w.count;
      break;
    }
    return w;
  };

  const int rank = CLUSTER ? blockIdx.x % ranks : 0;
  if (CLUSTER && threadIdx.x == 0) {
    // this CTA's share of its block's tiles
    const int unit = blockIdx.x / ranks, r = unit / (most_blocks * p.Hkv), rem = unit % (most_blocks * p.Hkv);
    Piece w;
    w.r = r, w.kvh = rem / most_blocks, w.tok0 = rem % most_blocks * tokens_per_block;
    w.q_begin = p.cu_q[r], w.kv_len = p.kv_lens[r];
    const int q_len = p.cu_q[r + 1] - w.q_begin;
    w.ctx = max(0, w.kv_len - q_len);
    w.lo = low_of(w.ctx), w.tile0 = w.lo / KT;
    w.nrows = max(0, min(tokens_per_block, q_len - w.tok0) * p.g);
    w.n = w.nrows > 0 ? tiles_of(q_len, w.kv_len) : 0;
    const int per = (w.n + ranks - 1) / ranks;
    w.first = min(w.n, rank * per), w.count = min(per, w.n - w.first);
    w.at = w.next = 0;
    mc.own = w;
  }
  if (CLUSTER) __syncthreads();
  // The tiles' copies, of keys or of values: the lanes look up the pages of several tiles in one round trip, a batch ahead; for a tile, lane i issues its
  // i-th page's.
  struct Lookup {
    int entry, ahead;
  };
  const int page_shift = __ffs(p.page_size) - 1;         // pages are a power of two of keys, 8 to 128
  const int pages_per_tile = KT >> page_shift, tiles_per_batch = 32 / pages_per_tile;
  auto look = [&](const Piece& w, int j) {               // this lane's page of the batch that begins with the piece's tile j
    const int key = (w.tile0 + w.first + j) * KT + lane * p.page_size, slot = key >> page_shift;
    // pages that hold a key some row reads, and exist
    return j < w.count && key < w.kv_len && key + p.page_size > w.lo && slot < p.table_width ? p.block_table[(size_t)w.r * p.table_width + slot] : -1;
  };
  auto copy = [&](const Piece& w, Lookup& u, int j, uint32_t to, uint64_t& bar, const CUtensorMap* map) {
    const int jb = j % tiles_per_batch;
    if (jb == 0 && j > 0) u.entry = u.ahead;
    if (jb == 0) u.ahead = look(w, j + tiles_per_batch);
    const int page = __shfl_sync(0xffffffffu, u.entry, (jb * pages_per_tile + lane) & 31);
    if (lane == 0) mbar_arrive_expect_tx(smem_u32(&bar), S::BYTES);
    __syncwarp();
    if (lane < pages_per_tile) {
#pragma unroll
      for (int h = 0; h < BLOCKS; ++h)
        tma_load_4d(to + h * BLOCK_BYTES + lane * p.page_size * ROW_BYTES, map, smem_u32(&bar), h * 64, 0, w.kvh, page);
    }
  };
  auto gave_up = [&](bool ran_out) {
    if (ran_out) gb_err::report(ERR_WAIT_EMPTY);
    *abort_s = 1;
    // wind down: the copies in flight need microseconds to land; two milliseconds before the shared memory is given up
    if (lane == 0) {
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {}
    }
  };
  if (warp == 0) {
    // ------------------------------------------------------------------ pieces, queries, keys
    int ks = 0, kpar = 1;             // the stage to fill and the phase of its "empty" barrier
    bool ok = true, ran_out = false;
    Piece w = CLUSTER ? mc.own : piece_at(a_begin);
    for (int it = 0; ok; ++it) {
      Lookup u{look(w, 0), -1};
      if (it > 0) ok = mbar_wait_warp(smem_u32(&mc.q_empty), (it - 1) & 1, abort_s, ran_out);
      if (!ok) break;
      if (lane == 0) {
        mc.piece[it & 1] = w;         // (who waits for the queries reads it behind that)
        if (w.count > 0) {
          mbar_arrive_expect_tx(smem_u32(&mc.q_full), (uint32_t)(box_tokens * p.g * ROW_BYTES * BLOCKS));
#pragma unroll
          for (int h = 0; h < BLOCKS; ++h)
            tma_load_3d(q_s + h * BLOCK_BYTES, &q_map, smem_u32(&mc.q_full), h * 64, w.kvh * p.g, w.q_begin + w.tok0);
        } else {
          mbar_arrive(smem_u32(&mc.q_full));
        }
      }
      __syncwarp();
      if (w.count == 0) break;
      for (int j = 0; j < w.count; ++j) {
        if (!(ok = mbar_wait_warp(smem_u32(&mc.k_empty[ks]), kpar, abort_s, ran_out))) break;
        copy(w, u, j, k_s + ks * S::BYTES, mc.k_full[ks], &k_map);
        if (++ks == K_STAGES) ks = 0, kpar ^= 1;
      }
      if (CLUSTER) w.count = 0;
      else w = piece_at(w.next);
    }
    if (!ok) gave_up(ran_out);
  } else if (warp == THREADS / 32 - 1) {
    // ------------------------------------------------------------------ values
    int vs = 0, vpar = 1;
    bool ok = true, ran_out = false;
    for (int it = 0; ok; ++it) {
      if (!(ok = mbar_wait_warp(smem_u32(&mc.q_full), it & 1, abort_s, ran_out))) break;
      const Piece w = mc.piece[it & 1];
      if (w.count == 0) break;
      // (The piece has been seen, and that its queries came. The softmax warps alone do not say so: a piece of one or two tiles has all its scores before any
      // of its values, and the barrier could be through the next piece's phase by the time that this warp looks at it.)
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&mc.q_empty));
      Lookup u{look(w, 0), -1};
      for (int j = 0; j < w.count; ++j) {
        if (!(ok = mbar_wait_warp(smem_u32(&mc.v_empty[vs]), vpar, abort_s, ran_out))) break;
        copy(w, u, j, v_s + vs * S::BYTES, mc.v_full[vs], &v_map);
        if (++vs == V_STAGES) vs = 0, vpar ^= 1;
      }
    }
    if (!ok) gave_up(ran_out);
  } else if (warp == 1) {
    // -------------------------------------------------------------------- MMA issuer
    // The S products run two tiles ahead of the P V products, across the pieces' borders. After a tile's softmax its P V goes first: it
    // reads the weights from the S buffer that the S product two tiles ahead then overwrites (products run in the order of their issue).
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = instr_desc_bf16(QROWS, KT), idesc_o = instr_desc_bf16(QROWS, HD) | INSTR_B_MN_MAJOR;
    const uint64_t dq0 = smem_desc_sw128(q_s), dk0 = smem_desc_sw128(k_s), dv0 = smem_desc_sw128_mn(v_s, BLOCKS > 1 ? BLOCK_BYTES : 16);
    bool ok = true, ran_out = false;
    int ks = 0, kpar = 0, vs = 0, vpar = 0, sb = 0, pb = 0, ppar = 0;
    auto wait_k = [&]() {
      if (ok) ok = mbar_wait_warp(smem_u32(&mc.k_full[ks]), kpar, abort_s, ran_out);
    };
    auto issue_s = [&]() {
      tc_fence_after_sync();
      if (leader) {
#pragma unroll
        for (int h = 0; h < BLOCKS; ++h)
          mma_bf16_x4(tmem_base + sb * KT, dq0 + (uint64_t)(h * (BLOCK_BYTES >> 4)), dk0 + (uint64_t)(ks * (S::BYTES >> 4) + h * (BLOCK_BYTES >> 4)),
                      idesc_s, 2, 2, h > 0);
        mma_commit(smem_u32(&mc.s_ready[sb]));
        if (S::KEYS_FREED_BY_COMMIT) mma_commit(smem_u32(&mc.k_empty[ks]));
      }
      __syncwarp();
      if (++ks == K_STAGES) ks = 0, kpar ^= 1;
      if (++sb == S_BUFS) sb = 0;
    };
    for (int it = 0; ok; ++it) {
      // (the next piece's first S products run while the softmax warps are at this one's end)
      if (!(ok = mbar_wait_warp(smem_u32(&mc.q_full), it & 1, abort_s, ran_out))) break;
      const int count = mc.piece[it & 1].count;
      if (count == 0) break;
      for (int j = 0; j < min(S_BUFS, count) && ok; ++j) {
        wait_k();
        if (ok) issue_s();
      }
      for (int j = 0; j < count && ok; ++j) {
        // (a wait costs near two hundred clocks even when there is nothing to wait for: those for keys and values go in front of the one for the weights)
        const bool more = j + S_BUFS < count;
        if (more) wait_k();
        if (ok) ok = mbar_wait_warp(smem_u32(&mc.v_full[vs]), vpar, abort_s, ran_out);
        if (ok) ok = mbar_wait_warp(smem_u32(&mc.p_ready[pb]), ppar, abort_s, ran_out);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
#pragma unroll
          for (int g = 0; g < GROUPS; ++g)
            mma_bf16_ts<GK / 16>(tmem_base + O_COL0 + g * HD, tmem_base + pb * KT + g * GK,
                                 dv0 + (uint64_t)(vs * (S::BYTES >> 4) + g * (GK * ROW_BYTES >> 4)), idesc_o, 16 * ROW_BYTES >> 4, j > 0);
          mma_commit(smem_u32(&mc.o_ready[pb]));
        }
        __syncwarp();
        if (more) issue_s();
        if (++vs == V_STAGES) vs = 0, vpar ^= 1;
        if (++pb == S_BUFS) pb = 0, ppar ^= 1;
      }
    }
    if (!ok) {
      if (ran_out) gb_err::report(ERR_WAIT_FULL);
      *abort_s = 1;
    }
  } else {
    // -------------------------------------------------------------------- softmax warps
    const int grp = (warp - 2) >> 2;
    const int quarter = warp & 3;                        // the TMEM lanes this warp may read
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_mine = lane_addr + O_COL0 + grp * HD;
    const float scale_log2 = p.scale * 1.4426950408889634f;
    bool ok = true;
    int gt = 0, it = 0, et = 0;   // tiles, pieces and masked tiles so far
    int sb = 0, sph = 0, kstage = 0, vstage = 0, vpar = 0, vfree = 0;       // (vfree: the stage of values to give back next)
    int freed = 0;                // tiles whose values have been given back
    const bool passes_on = threadIdx.x == 64;      // one thread tells the TMA warp what the tensor core has finished with
    auto wait = [&](uint64_t& bar, int parity, int code) {       // the whole warp's: it stays together
      bool ran_out;
      if (!mbar_wait_warp(smem_u32(&bar), parity, abort_s, ran_out)) {
        if (ran_out) gb_err::report(code);
        ok = false;
        *abort_s = 1;
      }
    };
    // Until the P V products of the tile counted t have ended. (Not asked for every tile: those of t - 2, the barrier's phase in front, have ended since the
    // scores of t were there, those of t + 2 wait for this warp.)
    auto wait_o = [&](int t) {
      wait(mc.o_ready[t & 1], t >> 1 & 1, ERR_WAIT_ACCUM);
      tc_fence_after_sync();
    };
    // All softmax warps meet, as at a barrier, but none waits for ever for one that has given up.
    int meetings = 0;
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&mc.met));
      wait(mc.met, meetings++ & 1, ERR_WAIT_DRAIN);
    };
    for (;; ++it) {
      wait(mc.q_full, it & 1, ERR_WAIT_FULL);        // (the piece; its queries have been waited for by the products)
      if (!ok) break;
      const Piece& w = mc.piece[it & 1];             // (read where it is used: registers are short)
      const int count = w.count;
      if (count == 0) break;
      const bool there = row < w.nrows;
      const bool active = quarter * 32 < w.nrows;        // this warp has a row
      // tiles from here on, and up to there, hold keys that some row does not read
      const int edge_from = w.ctx, edge_to = p.window > 0 ? w.kv_len - p.window : 0, first_key = (w.tile0 + w.first) * KT;
      float m = -INFINITY, l = 0.f;      // m: the reference maximum of the raw dot products
      bool spoiled = false;              // this row reads a value that is not finite

      for (int j = 0; j < count && ok; ++j, ++gt) {
        // (What an edge asks of the row is read while the scores are made.)
        const int tile_key0 = first_key + j * KT, key0 = tile_key0 + grp * GK;
        const bool edge = tile_key0 + KT > edge_from || tile_key0 < edge_to;
        unsigned long long sees = ~0ull;
        if (edge) {
          const int token = w.q_begin + w.tok0 + (there ? row / p.g : 0);
          // the keys of these 64 that the row reads: context, then drafted tokens by their bits
          const int c = w.ctx - key0;
          sees = 0;
          if (there) {
            const uint32_t* bits = p.mask + (size_t)token * p.mask_words;
            if (c > 0) {
              const int row_start = p.window > 0 ? max(0, p.positions[token] + 1 - p.window) : 0;
              sees = c >= 64 ? ~0ull : (1ull << c) - 1;
              const int s0 = row_start - key0;
              if (s0 > 0) sees &= s0 >= 64 ? 0ull : ~0ull << s0;
            }
            if (c < 64) {
              const int from = max(0, -c), word = from >> 5;
              auto at = [&](int i) -> unsigned long long { return i < p.mask_words ? bits[i] : 0u; };
              unsigned long long b = at(word) | (at(word + 1) << 32);
              if (from & 31) b = (b >> (from & 31)) | (at(word + 2) << (64 - (from & 31)));
              const int left = w.kv_len - key0 - max(0, c);         // drafted tokens from there on
              b &= left >= 64 ? ~0ull : left > 0 ? (1ull << left) - 1 : 0ull;
              sees |= c > 0 ? b << c : b;
            }
          }
        }
        // The values of a tile at an edge: rows that nobody may read are cleared, those that are not finite noted.
        auto look = [&]() {
          if (!edge) return;
          wait(mc.v_full[vstage], vpar, ERR_WAIT_FULL);
          bool bad = false;
          if (ok && row < GK) {               // (a row of values to each of half of the group's threads)
            const int vrow = grp * GK + row, key = tile_key0 + vrow;
            const uint32_t vaddr = v_s + vstage * S::BYTES + vrow * ROW_BYTES;
            bool clear = key < w.lo || key >= w.kv_len;
            if (!clear) {
              bool odd = false;
#pragma unroll
              for (int c = 0; c < BLOCKS * (ROW_BYTES / 16); ++c) {
                // (from a chunk of its own on: 32 rows' chunks at the same place share four banks)
                const uint4 x = ld_shared_v4(vaddr + (c / 8) * BLOCK_BYTES + ((c + row) & 7) * 16);
                odd = odd || not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
              }
              clear = bad = odd;
            }
            if (clear) {
#pragma unroll
              for (int c = 0; c < BLOCKS * (ROW_BYTES / 16); ++c) clear_shared_v4(vaddr + (c / 8) * BLOCK_BYTES + ((c + row) & 7) * 16);
            }
            fence_proxy_async();            // the tensor core reads the values through the async proxy
          }
          const uint32_t bads = __ballot_sync(0xffffffffu, bad);
          if (quarter < 2 && lane == 0) mc.bad[et & 1][grp][quarter] = bads;
          // (All four warps arrive, those too that look at no value: so none is two such tiles in front of another, whose wait would take the phase after
          // the next for its own, and whose notes would be written over.)
          if (lane == 0) mbar_arrive(smem_u32(&mc.looked[grp]));
          wait(mc.looked[grp], et & 1, ERR_WAIT_FULL);
          const unsigned long long spoils = mc.bad[et & 1][grp][0] | ((unsigned long long)mc.bad[et & 1][grp][1] << 32);
          ++et;
          spoiled = spoiled || (sees & spoils) != 0;
        };
        // (In front of the scores if the tile is one of few: then the values come no later than the keys. Their stage was given back before the scores in
        // front were used, so that they come whatever this warp waits for.)
        if (CLUSTER) look();
        wait(mc.s_ready[sb], sph, ERR_WAIT_ACCUM);
        if (!ok) break;
        tc_fence_after_sync();
        // S of this tile is complete: its keys have been read, after a piece's last tile its queries (every warp says so, and the values' once it has seen the
        // piece: it is done with the piece in front), and the values of the tile two in front (products run in the order of their issue)
        if (j == count - 1 && lane == 0) mbar_arrive(smem_u32(&mc.q_empty));
        if (passes_on) {
          if (freed < gt - 1) {
            mbar_arrive(smem_u32(&mc.v_empty[vfree]));
            if (++vfree == V_STAGES) vfree = 0;
            ++freed;
          }
          if (!S::KEYS_FREED_BY_COMMIT) mbar_arrive(smem_u32(&mc.k_empty[kstage]));
        }
        if (++kstage == K_STAGES) kstage = 0;
        const uint32_t s_addr = lane_addr + sb * KT + grp * GK;
        uint32_t sv[GK / 32][32];
        if (active) {
#pragma unroll
          for (int h = 0; h < GK / 32; ++h) tmem_ld_32(s_addr + h * 32, sv[h]);
        }
        if (!CLUSTER) look();
        if (++vstage == V_STAGES) vstage = 0, vpar ^= 1;
        if (!ok) break;
        if (active) {
          tmem_ld_wait();
          auto sc = [&](int ch) -> float& { return reinterpret_cast<float&>(sv[ch >> 5][ch & 31]); };
          if (edge) {
            const uint32_t half[2] = {(uint32_t)sees, (uint32_t)(sees >> 32)};
#pragma unroll
            for (int ch = 0; ch < GK; ++ch)
              if (!(half[ch >> 5] >> (ch & 31) & 1u)) sc(ch) = -INFINITY;
          }
          float mx[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int ch = 0; ch < GK; ch += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], sc(ch + e), sc(ch + 4 + e));
          }
          const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          // The reference moves only if some row of the warp has outgrown it by more than 2^8; then the warp rescales what it has accumulated.
          // (Lanes without a row hold whatever was in shared memory: they have no say.)
          const bool grown = there && m != -INFINITY && (m_new - m) * scale_log2 > RESCALE_ABOVE;
          if (j > 0 && __any_sync(0xffffffffu, grown)) {
            wait_o(gt - 1);
            if (ok) {
              const float corr = m == -INFINITY ? 1.f : fast_exp2((m - m_new) * scale_log2);
#pragma unroll
              for (int h = 0; h < HD / 32; ++h) {
                uint32_t v[32];
                tmem_ld_32(o_mine + h * 32, v);
                tmem_ld_wait();
#pragma unroll
                for (int ch = 0; ch < 32; ++ch) v[ch] = __float_as_uint(__uint_as_float(v[ch]) * corr);
                tmem_st_32(o_mine + h * 32, v);
              }
              l *= corr;
              m = m_new;
            }
          } else if (m == -INFINITY) {
            m = m_new;
          }
          const float neg_m = m == -INFINITY ? 0.f : -m * scale_log2;       // nothing valid yet: avoid inf - inf
          const Two scale_two = two(scale_log2, scale_log2), neg_m_two = two(neg_m, neg_m);
          Two ls[4] = {two(0.f, 0.f), two(0.f, 0.f), two(0.f, 0.f), two(0.f, 0.f)};
          uint32_t pk[GK / 2];
#pragma unroll
          for (int ch = 0; ch < GK; ch += 2) {
            const float2 x = apart(fma_two(two(sc(ch), sc(ch + 1)), scale_two, neg_m_two));
            const float wx = fast_exp2(x.x), wy = fast_exp2(x.y);
            ls[(ch >> 1) & 3] = add_two(ls[(ch >> 1) & 3], two(wx, wy));
            // Weights are rounded to bfloat16, the type of the values that they multiply: half a step of 2^-8 each, averaged out by the
            // sum over keys; the denominator takes them as they are.
            pk[ch >> 1] = pack_bf16(wx, wy);
          }
          const float2 sums = apart(add_two(add_two(ls[0], ls[1]), add_two(ls[2], ls[3])));
          l += sums.x + sums.y;
          tmem_st(s_addr, pk);            // over the first half of the scores just read
          tmem_st_wait();
        }
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&mc.p_ready[sb]));
        if (++sb == S_BUFS) sb = 0, sph ^= 1;
      }
      if (ok) {
        wait_o(gt - 1);
        for (; passes_on && ok && freed < gt; ++freed) {
          mbar_arrive(smem_u32(&mc.v_empty[vfree]));
          if (++vfree == V_STAGES) vfree = 0;
        }
      }
      const int token = w.q_begin + w.tok0 + (there ? row / p.g : 0);
      // ---- merge the groups: each has its share of the channels, summed over both accumulators
      const int mb = it & 1;
      if (spoiled) l = NAN;
      mc.ml[mb][grp][row] = make_float2(m, l);
      tc_fence_before_sync();
      meet();
      tc_fence_after_sync();
      const bool whole = !CLUSTER && w.count == w.n;
      const int c0 = CLUSTER ? 0 : w.at / stretch, c1 = CLUSTER ? 0 : (w.at + w.n - 1) / stretch;           // the CTAs that have the block's first and last tile
      // (CLUSTER: where queries, keys and values were, which have all been used)
      float* const part = CLUSTER ? reinterpret_cast<float*>(smem_raw) : parts + ((size_t)blockIdx.x * 2 + ((int)blockIdx.x == c0 ? 1 : 0)) * S::PART_FLOATS;
      if (ok && !*abort_s && active) {
        float mt = -INFINITY, lt = 0.f, f[GROUPS];
        float2 x[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) x[g] = mc.ml[mb][g][row], mt = fmaxf(mt, x[g].x);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          // (a stream without a key: its accumulator means nothing, -inf stands for that; without a number: it has no reference. One whose weights are nothing beside
          // the other's counts with them: what is not finite in it stays so)
          f[g] = x[g].x == -INFINITY ? (x[g].y == 0.f ? -INFINITY : NAN) : fast_exp2((x[g].x - mt) * scale_log2);
          lt += x[g].x == -INFINITY ? x[g].y : x[g].y * f[g];
        }
        const float inv = whole ? (lt == 0.f ? 0.f : 1.0f / lt) : 1.f;
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) +
                             ((size_t)token * p.Hq + w.kvh * p.g + (there ? row % p.g : 0)) * HD + grp * CH;
        float4* pdst = reinterpret_cast<float4*>(part) + grp * (CH / 4) * QROWS + row;        // [HD / 4][rows]: neighbouring lanes side by side
#pragma unroll
        for (int h = 0; h < CH / 16; ++h) {
          float t[16];
          uint32_t v[2][16];
          tmem_ld_16(lane_addr + O_COL0 + grp * CH + h * 16, v[0]);
          tmem_ld_16(lane_addr + O_COL0 + HD + grp * CH + h * 16, v[1]);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            t[e] = f[0] == -INFINITY ? 0.f : __uint_as_float(v[0][e]) * (f[0] * inv);
            t[e] += f[1] == -INFINITY ? 0.f : __uint_as_float(v[1][e]) * (f[1] * inv);
          }
          if (there) {
            if (whole) {
              uint4 w0, w1;
              w0.x = pack_bf16(t[0], t[1]), w0.y = pack_bf16(t[2], t[3]), w0.z = pack_bf16(t[4], t[5]), w0.w = pack_bf16(t[6], t[7]);
              w1.x = pack_bf16(t[8], t[9]), w1.y = pack_bf16(t[10], t[11]), w1.z = pack_bf16(t[12], t[13]), w1.w = pack_bf16(t[14], t[15]);
              *reinterpret_cast<uint4*>(dst + h * 16) = w0;
              *reinterpret_cast<uint4*>(dst + h * 16 + 8) = w1;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) pdst[(h * 4 + e) * QROWS] = make_float4(t[4 * e], t[4 * e + 1], t[4 * e + 2], t[4 * e + 3]);
            }
          }
        }
        if (there && !whole && grp == 0)
          *reinterpret_cast<float2*>(part + QROWS * HD + row * 2) = make_float2(mt * scale_log2, lt);       // (the scale is positive)
      }
      tc_fence_before_sync();
      if (!CLUSTER && !whole) {
        // ---- the CTA that counts the last of the block's pieces joins them, in the order of the keys. (A CTA that gave up counts too: the
        // error word says that the results are not to be trusted.)
        // (The meeting orders what the CTA has written in front of the count, which is a release, and behind it what it reads of the others'.)
        meet();
        if (threadIdx.x == 64) {
          int seen;
          asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counters + c0) : "memory");
          mc.last = seen == c1 - c0;
          if (seen == c1 - c0) counters[c0] = 0;         // as the next launch expects it
        }
        meet();
        if (ok && mc.last) {
          join_pieces<HD>(parts, c0, c1, w.nrows, reinterpret_cast<__nv_bfloat16*>(p.out) + (((size_t)w.q_begin + w.tok0) * p.Hq + w.kvh * p.g) * HD, p.g,
                          p.Hq);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (CLUSTER) {
    // ---- the CTAs of the cluster share the rows out, and read the pieces' sums from one another
    float* const part = reinterpret_cast<float*>(smem_raw);
    const Piece& w = mc.own;
    if (w.count == 0)
      for (int i = threadIdx.x; i < QROWS; i += THREADS) reinterpret_cast<float2*>(part + QROWS * HD)[i] = make_float2(-INFINITY, 0.f);
    cluster_arrive_wait();
    const int items = w.nrows * (HD / 8), mine = (items + ranks - 1) / ranks;          // eight channels of a row
    for (int i = rank * mine + threadIdx.x; i < min(items, (rank + 1) * mine) && !*abort_s; i += THREADS) {
      const int row = i % w.nrows, f0 = i / w.nrows * 2;
      const uint32_t ml_at = smem_u32(part + QROWS * HD + row * 2), v_at = smem_u32(part) + (uint32_t)(f0 * QROWS + row) * 16;
      Join<2> join;
#pragma unroll 1
      for (int q = 0; q < ranks; q += 4) {
        float2 ml[4];
        float4 v[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t from = min(q + u, ranks - 1);
          ml[u] = ld_cluster_f2(map_to_rank(ml_at, from));
          v[u][0] = ld_cluster_f4(map_to_rank(v_at, from));
          v[u][1] = ld_cluster_f4(map_to_rank(v_at + QROWS * 16, from));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (q + u < ranks) join.add(ml[u], v[u]);
      }
      join.store(reinterpret_cast<__nv_bfloat16*>(p.out) +
                 ((size_t)(w.q_begin + w.tok0 + row / p.g) * p.Hq + w.kvh * p.g + row % p.g) * HD + f0 * 4);
    }
    cluster_read_wait();                               // nobody leaves while another reads
  }
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// ------------------------------------------------------------------ host side
// A tensor [d3][d2][d1][hd] of bfloat16 (channels contiguous) through boxes [1][b2][b1][64] (d3 = 0: three dimensions), 128-byte
// swizzle; what lies outside reads as zeros.
int tensor_map(const void* ptr, int hd, long long d1, long long d2, long long d3, int b1, int b2, CUtensorMap* out) {
  tc_host::EncodeTiledFn fn = tc_host::encode_fn();
  if (!fn) return gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled is not available from this driver");
  const int rank = d3 > 0 ? 4 : 3;
  cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)d1, (cuuint64_t)d2, (cuuint64_t)(d3 > 0 ? d3 : 1)};
  cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)hd * 2 * d1, (cuuint64_t)hd * 2 * d1 * d2};
  cuuint32_t box[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(ptr), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? GB_OK : gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled failed with code %d for an attention operand", (int)r);
}

// CTAs of a cluster that share the keys of each of `units` blocks of rows, or 0: stretches. Clusters need no scratch memory, no scan of the lengths, and
// join faster (a request of 8 tokens, 8 heads of 128, 500 keys: 9.2 us against 13.3; 8,000 keys: 16.5 against 22), but they are of 2, 4 or 8 CTAs (16 took
// twice as long: hardly any run at once), so that SMs stay idle, and wait for the longest request (32,000 keys: 46 against 38). In microseconds, with what both
// have in common left out: a tile takes 1.1, a piece of a stretch 0.4 to join.
template <int HD>
int cluster_ranks(long long units, int tiles, int sms, int smem) {
  static branches::AskedOnce<4> most;                            // clusters of 2^i CTAs that run at once
  const float stretch = (float)((units * (tiles + BLOCK_COST) + sms - 1) / sms < MIN_STRETCH ? MIN_STRETCH : (units * (tiles + BLOCK_COST) + sms - 1) / sms);
  float best = 3.f + 1.1f * stretch + 0.4f * (tiles / stretch);
  int ranks = 0;
  for (int i = 1; i <= 3; ++i) {
    const int room = most.get(i, [&] {
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3(1 << i), config.blockDim = dim3(THREADS), config.dynamicSmemBytes = smem;
      cudaLaunchAttribute shape;
      shape.id = cudaLaunchAttributeClusterDimension;
      shape.val.clusterDim.x = 1 << i, shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
      config.attrs = &shape, config.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, attention_tree_tc_kernel<HD, true>, &config) != cudaSuccess) n = 0, cudaGetLastError();
      return n;
    });
    const float time = 1.1f * ((tiles + (1 << i) - 1) >> i);
    if (units <= room && time < best) best = time, ranks = 1 << i;
  }
  return ranks;
}

template <int HD>
int launch(const TreeParams& whole, int max_q_len, int max_kv_len, int* counters, float* parts, cudaStream_t stream) {
  using S = Shape<HD>;
  CUtensorMap qm, km, vm;
  const int tokens_per_block = QROWS / whole.g, box_tokens = tokens_per_block < max_q_len ? tokens_per_block : max_q_len;
  int rc = tensor_map(whole.q, HD, whole.Hq, whole.T, 0, whole.g, box_tokens, &qm);
  if (!rc) rc = tensor_map(whole.k_pool, HD, whole.page_size, whole.Hkv, whole.pages, whole.page_size, 1, &km);
  if (!rc) rc = tensor_map(whole.v_pool, HD, whole.page_size, whole.Hkv, whole.pages, whole.page_size, 1, &vm);
  if (rc) return rc;
  const int sms = tc_host::sm_count();
  const auto smem = [](int R) { return S::TILE_BYTES + (int)sizeof(Misc) + 4 * (3 * R + 2); };
  static_assert(S::TILE_BYTES + (int)sizeof(Misc) + 4 * (3 * MAX_REQUESTS + 2) <= 232448, "shared memory of one CTA");
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    cudaError_t e = cudaFuncSetAttribute(attention_tree_tc_kernel<HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem(MAX_REQUESTS));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_tree_tc_kernel<HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem(0));
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "tree_attention: %s", cudaGetErrorString(e));
    configured.done();
  }
  const int blocks = (max_q_len + tokens_per_block - 1) / tokens_per_block, tiles = max_kv_len / KT + 1;
  const long long units = (long long)whole.R * whole.Hkv * blocks;
  const int ranks = cluster_ranks<HD>(units, tiles, sms, smem(0));
  if (ranks > 0)
    return gb::check_pdl_launch(gb::launch_pdl(attention_tree_tc_kernel<HD, true>, dim3((unsigned)units * ranks), dim3(THREADS), smem(0), stream,
                                               dim3(ranks, 1, 1), qm, km, vm, whole, box_tokens, 0, ranks, blocks, parts, counters), "tree_attention");
  for (int r0 = 0; r0 < whole.R; r0 += MAX_REQUESTS) {
    TreeParams p = whole;
    p.R = whole.R - r0 < MAX_REQUESTS ? whole.R - r0 : MAX_REQUESTS;
    p.cu_q += r0, p.kv_lens += r0, p.block_table += (size_t)r0 * p.table_width;
    rc = gb::check_pdl_launch(gb::launch_pdl(attention_tree_tc_kernel<HD, false>, dim3(sms < COUNTERS ? sms : COUNTERS), dim3(THREADS), smem(p.R), stream,
                                             dim3(1, 1, 1), qm, km, vm, p, box_tokens, MIN_STRETCH, 0, 0, parts, counters), "tree_attention");
    if (rc) return rc;
  }
  return GB_OK;
}

}  // namespace

// Bytes of scratch memory and of counters a call needs; the counters are zero before the first one, and every call leaves them zero.
GB_EXPORT long long gb_tree_attention_scratch_bytes(int head_dim, long long* counter_bytes) {
  *counter_bytes = 4ll * COUNTERS;
  return 2ll * tc_host::sm_count() * QROWS * (head_dim + 2) * 4;
}

GB_EXPORT int gb_tree_attention_tc(const branches::TreeCall* call) {
  const TreeParams p = call->params();
  int* counters = reinterpret_cast<int*>(call->counters);
  float* parts = reinterpret_cast<float*>(call->scratch);
  const int max_q_len = (int)call->max_q_len, max_kv_len = (int)call->max_kv_len;
  if (call->head_dim == 64) return launch<64>(p, max_q_len, max_kv_len, counters, parts, (cudaStream_t)call->stream);
  if (call->head_dim == 128) return launch<128>(p, max_q_len, max_kv_len, counters, parts, (cudaStream_t)call->stream);
  return gb::fail(GB_UNSUPPORTED, "tree_attention: head size %lld", call->head_dim);
}

GB_EXPORT int gb_tree_attention_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_tree_attention_set_error_sink(int* host_word) { return gb_err::set_sink(host_word); }
