// Attention of single tokens (few query rows a request) over pages of E4M3 codes with a scale per page and head.
//
//   s_j = (q . k8_j) * ks(page of j) * scale over keys [start, pos];  out = sum_j softmax(s)_j vs(page of j) v8_j
// (garuda/src/llama/mod.rs:793-818; the window garuda/src/cache/mod.rs:333-338; query head h reads key/value head h / g).
//
// Bound by the stream of codes, 2 * HD bytes a key and head, so they go from shared memory into the matrix instructions as they are
// (tcgen05.mma kind f8f6f4, 32-bit sums), and what has more than four bits is split instead: a query row, scaled by a power of two to a largest
// of at most 448, is the sum of an E4M3 row and 1/16 of another (a bfloat16's eight bits are four and four: exact down to 2^-13 of the
// row's largest; what is below that loses bits, and is gone below 2^-21), and a weight exp(s) * vs is three codes, the second and third in units of 1/32 and 1/1024: twelve
// bits, down to 2^-24 of the reference. (Groups of more than eight heads: two codes, nine bits, down to 2^-22, and a reference that
// follows every larger one.) Products of one tile of 128 keys:
//   S^T [128 keys, N] = K [128, HD] * Q [N, HD]^T         N = 16 (or 32): the rows' codes, then what these leave
//   O [rows, HD]     += P [rows, 128] * V [128, HD]       P's rows: the weights' first codes, then the others; V as it lies, keys along its
//                                                         rows. The products' other rows (128 in all) read whatever lies behind P, and
//                                                         nobody reads their sums
// A thread has a key: its N sums from tensor memory are its scores with all rows, so the 128 threads share out the exponentials evenly, and
// what is per key (page, scales, mask) is per thread. (mma.sync on E4M3 takes 860 instructions for 32 keys, as this hardware has no
// such product and converts; with the codes converted to halves by hand 700; both were bound by instructions at 5.0 TB/s and below. Here
// 128 keys take some 500.) Maxima and denominators are 32-bit.
//
// Scales cost nothing per key: ks goes into the score's factor, vs, as a power of two, is added to the score, and the denominator takes it out
// again. So what weights refer to is a row's own largest exp(s) * vs: a page that a row may not read, or whose keys have no weight,
// takes no bits from the others however large its values are (with the largest vs of all pages in the reference, weights of pages
// 2^-20 below it were off by several per cent, below 2^-25 gone). The reference is common to the tile's 128 keys. It follows the
// running maximum only when some key exceeds it by more than 2^3 (a vote a tile; following at once cost 0.8 us a time, some 14 times in 60
// tiles), and then the sums in tensor memory are brought to it.
//
// Work: the tiles of all requests and heads in a row, an equal stretch to every CTA, so that requests of unequal length do not wait for
// the longest; a request that falls to several CTAs is merged by the one that finishes last, in their order, from scratch memory, so
// that results do not depend on who that is. Within a CTA, the copies, the scores' products and the queries of the next request's head
// run ahead across the border.
//   warp 0     TMA: a box a page (swizzled) into a ring of stages; looks up pages and scales four tiles at a time, two steps ahead
//   warp 1     one elected lane issues the products: S^T of a tile, then O += P V of the tile before
//   warps 2-5  scores, maxima, weights; the next head's queries as codes; results
// Two CTAs an SM (N = 16; one with N = 32). Every wait is bounded.
// Few short heads (CLUSTER): one head to a thread-block cluster, whose CTAs share its tiles and store their rows of sums into the shared
// memory of the first, which adds them up in the CTAs' order behind a barrier of the cluster. (Asynchronous stores counted on a barrier in
// memory took 2 us for 400 of them.) 4 requests of 65,536 positions, 8 heads of 128: 5.9 TB/s from a graph (5.4 a call from Python); one of 500: 7.1 us; 8 of 2,048, 4 of 64: 11.0.
#include "attention_float8.cuh"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

#include <algorithm>
#include <type_traits>

namespace {

using namespace tc;
using namespace attn8;

constexpr int KT = 128;                 // keys per tile
constexpr int THREADS = 192;
constexpr int MAX_ROWS = 16;
constexpr int MAX_CLUSTER = 8;
constexpr int SEGMENT = 4;              // what a request's head costs beside its tiles, in tiles (64 ragged requests: 2 129 us, 3 114, 4 109)
constexpr uint32_t O_COL = 64, TMEM_COLS = 256;          // tensor memory: two buffers of S^T, then O

template <int HD, int N, bool CLUSTER>
struct Shape {
  static constexpr int ROWS = N / 2;                                    // query rows
  static constexpr int OPERAND = KT * HD, STAGE = 2 * OPERAND;          // bytes: keys, values
  static constexpr int CTAS = N == 16 && !CLUSTER ? 2 : 1;              // per SM
  static constexpr int STAGES = (CLUSTER ? 128 : 192 / CTAS) * 1024 / STAGE;        // 3 (6, 4) of 32 KB, 6 (12, 8) of 16 KB
  static constexpr int PARTS = N == 16 ? 3 : 2;                         // codes of a weight
  // weights go to 2^GROWTH of the reference and are multiplied by 2^UP: codes go to 448
  static constexpr float GROWTH = PARTS == 3 ? 3.f : 0.f, UP = PARTS == 3 ? 5.f : 8.f;
  static constexpr int P_BYTES = PARTS * ROWS * KT, Q_BYTES = N * 128;
  static constexpr int RING_AT = 2 * P_BYTES + 2 * Q_BYTES;
  // CLUSTER: behind the ring the rows' sums, maxima and denominators of the cluster's CTAs, in its first
  static constexpr int RC = HD + 4, PARTS_AT = RING_AT + STAGES * STAGE;
  static constexpr int BYTES = PARTS_AT + (CLUSTER ? MAX_CLUSTER * ROWS * RC * 4 : 0);
  static constexpr int RS = HD + 2;                                     // a row's sums, maximum, denominator: a part in scratch memory
  static_assert(RING_AT % 1024 == 0 && P_BYTES + KT * 128 <= BYTES, "swizzled tiles; P's 128 rows end inside");
};

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[N]);
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t addr, uint32_t (&r)[16]) { tmem_ld_16(addr, r); }
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t addr, uint32_t (&r)[32]) { tmem_ld_32(addr, r); }

// x * 2^d, d <= 0, where 2^d by itself may be too small for a number in 32 bits.
__device__ __forceinline__ float times_power(float x, float d) {
  const float most = fmaxf(d, -120.f);
  return x * exp2_fast(most) * exp2_fast(d - most);
}
// Two weights as a code, 32 times what that leaves as a code, and (PARTS 3) 32 times what that leaves; in the low byte the first's.
template <int PARTS>
__device__ __forceinline__ void split(float a, float b, uint32_t (&code)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const uint16_t h = f8::encode2(a, b);
    code[i] = h;
    if (i + 1 < PARTS) {
      const float2 back = f8::decode2(h);
      a = (a - back.x) * 32.f, b = (b - back.y) * 32.f;
    }
  }
}
__device__ __forceinline__ void st_shared_u8(uint32_t addr, uint32_t v) { asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// Barrier of the four softmax warps; true for all if `mine` is for one.
__device__ __forceinline__ bool any_of_four(bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"((uint32_t)mine) : "memory");
  return r != 0;
}
// Into another CTA of the cluster.
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// The largest of a warp's (of those that are numbers).
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void sync_four() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

struct Bars {
  uint64_t full[12], empty[12], s_ready[2], p_ready[2], pv_done[2], q_ready[2], o_free;
  uint32_t tmem_base;
  int abort, last[2];
  int2 total, scan[6];
  float2 scales[12][8];            // a stage's ks of each sixteen keys (negative: no page there) and log2 of vs
  float factor[2][MAX_ROWS];       // per row of a head's queries: 2^e * scale * log2(e)
  float top[4][MAX_ROWS], corr[MAX_ROWS], vtop[4], lsum[4][MAX_ROWS];
};

// CLUSTER: one request's head per thread-block cluster, its CTAs share the tiles and merge through distributed shared memory.
template <int HD, int N, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, Shape<HD, N, CLUSTER>::CTAS)
attention_f8_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Params p,
                           const int min_tiles,        // (CLUSTER: CTAs of a cluster)
                           float* __restrict__ partials, int* __restrict__ counters) {
  using S = Shape<HD, N, CLUSTER>;
  constexpr int RS = S::RS, ROWS = S::ROWS, STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  uint8_t* const base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const uint32_t p_at = smem_u32(base), q_at = p_at + 2 * S::P_BYTES, ring = p_at + S::RING_AT;
  int* const cum = reinterpret_cast<int*>(base + S::BYTES);            // [R + 1]: tiles of a head of the requests in front
  int* const cost = cum + p.R + 1;                                     // [R + 1]: the same with SEGMENT more for every request with tiles
  int* const begin_s = cost + p.R + 1;                                 // [R + 1]: cu_q
  int* const len_s = begin_s + p.R + 1;                                // [R]: kv_lens

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&bars.full[s]), 2), mbar_init(smem_u32(&bars.empty[s]), 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bars.s_ready[b]), 1);
      mbar_init(smem_u32(&bars.p_ready[b]), 128);
      mbar_init(smem_u32(&bars.pv_done[b]), 1);
      mbar_init(smem_u32(&bars.q_ready[b]), 128);
    }
    mbar_init(smem_u32(&bars.o_free), 32);
    bars.abort = 0, bars.total = make_int2(0, 0);
    fence_barrier_init();
    fence_proxy_async();
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars.tmem_base), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars.tmem_base;
  volatile int* aborted = &bars.abort;
  gb::pdl_launch_dependents();
  if (CLUSTER) cluster_arrive_wait();      // the first CTA is there before sums are sent to it

  // ---- every request's tiles (the batch's lengths are there before the step's first kernel)
  struct Span {
    int lo, hi, pos0, nrows, q_begin;      // first and last key that any row reads
  };
  auto span_of = [&](int q_begin, int q_end, int kv_len) {
    Span s;
    s.q_begin = q_begin, s.nrows = (q_end - q_begin) * p.g, s.pos0 = kv_len - (q_end - q_begin);
    s.lo = p.window > 0 ? max(0, s.pos0 + 1 - p.window) : 0;
    s.hi = kv_len - 1;
    return s;
  };
  for (int r0 = 0; !CLUSTER && r0 < p.R; r0 += THREADS) {
    const int r = r0 + threadIdx.x;
    int n = 0;
    if (r < p.R) {
      const int q0 = p.cu_q[r], q1 = p.cu_q[r + 1], kv = p.kv_lens[r];
      begin_s[r] = q0, len_s[r] = kv;
      if (r + 1 == p.R) begin_s[r + 1] = q1;
      const Span s = span_of(q0, q1, kv);
      if (s.nrows > 0 && s.nrows <= ROWS && s.hi >= s.lo) n = s.hi / KT - s.lo / KT + 1;
    }
    int2 inc = make_int2(n, n > 0 ? 1 : 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc.x, o), v = __shfl_up_sync(0xffffffffu, inc.y, o);
      if (lane >= o) inc.x += u, inc.y += v;
    }
    if (lane == 31) bars.scan[warp] = inc;
    __syncthreads();
    int2 before = bars.total;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w)
      if (w < warp) before.x += bars.scan[w].x, before.y += bars.scan[w].y;
    before.x += inc.x, before.y += inc.y;          // with this request
    if (r < p.R) {
      cum[r] = before.x - n, cost[r] = before.x - n + SEGMENT * (before.y - (n > 0 ? 1 : 0));
      if (r + 1 == p.R) cum[r + 1] = before.x, cost[r + 1] = before.x + SEGMENT * before.y;
    }
    __syncthreads();
    if (threadIdx.x == THREADS - 1) bars.total = before;
    __syncthreads();
  }
  // Stretches are equal in cost: a request's head is its tiles and SEGMENT behind them. (The host has seen that all of it fits 31 bits.)
  const int tiles = CLUSTER ? 0 : cum[p.R] * p.Hkv, costs = CLUSTER ? 0 : cost[p.R] * p.Hkv;
  // as many workers as leave each min_tiles or so, and one for every head that has tiles
  const int workers = max(1, min((int)gridDim.x, max(tiles / min_tiles, bars.total.y * p.Hkv)));
  const int stretch = max(1, (costs + workers - 1) / workers);
  const int cta = blockIdx.x;
  auto find = [&](const int* sums, int at) {           // the last request whose heads begin at or before it
    int lo = 0, hi = p.R;
    while (hi - lo > 1) {              // (of requests without tiles at the same place the last one: it has some)
      const int mid = (lo + hi) >> 1;
      if (sums[mid] * p.Hkv <= at) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto begins_at = [&](int w) {                        // the first tile of worker w's stretch, in the row of all tiles
    const int c = w * stretch;
    if (c >= costs) return tiles;
    const int r = find(cost, c), n = cum[r + 1] - cum[r], rem = c - cost[r] * p.Hkv, head = rem / (n + SEGMENT);
    return cum[r] * p.Hkv + head * n + min(rem - head * (n + SEGMENT), n);
  };
  // CLUSTER: this CTA's head, its request's keys, and the CTA's part of them
  const int head = cta / min_tiles, rank = cta % min_tiles, own_r = head / p.Hkv;
  Span own{};
  int own_n = 0, own_per = 0;
  if (CLUSTER) {
    own = span_of(p.cu_q[own_r], p.cu_q[own_r + 1], p.kv_lens[own_r]);
    if (own.nrows > 0 && own.nrows <= ROWS && own.hi >= own.lo) own_n = own.hi / KT - own.lo / KT + 1;
    own_per = (own_n + min_tiles - 1) / min_tiles;
  }
  const int own_first = min(own_n, rank * own_per), own_end = min(own_n, own_first + own_per);
  const int a_begin = CLUSTER ? own_first : cta < workers ? begins_at(cta) : tiles;
  const int a_end = CLUSTER ? own_end : cta < workers ? begins_at(cta + 1) : tiles;
  const int my_tiles = a_end - a_begin;

  // A segment: one request's head, or this CTA's part of it: tiles first .. first + count of its n
  struct Segment {
    int r, kvh, first, n, count;
  };
  auto segment_at = [&](int a) {
    Segment g;
    if (CLUSTER) return Segment{own_r, head % p.Hkv, a, own_n, a_end - a};
    const int lo = find(cum, a);
    g.r = lo, g.n = cum[lo + 1] - cum[lo];
    const int rem = a - cum[lo] * p.Hkv;
    g.kvh = rem / g.n, g.first = rem % g.n;
    g.count = min(g.n - g.first, a_end - a);
    return g;
  };
  auto span_at = [&](int r) { return CLUSTER ? own : span_of(begin_s[r], begin_s[r + 1], len_s[r]); };

  // Everything else comes from the kernels in front, the pages among it: a page that this step writes is encoded again.
  gb::pdl_wait();

  if (my_tiles > 0 && warp == 0) {
    // ---------------------------------------------------------------- copies
    // Lane i looks up sixteen keys: block i % 8 of tile i / 8 of four.
    struct Lookup {
      int head, key, r, page;      // (r < 0: no tile)
      float ks, vs;
    } now{}, ahead{};
    const int sub = lane & 7, per_page = p.page >> 4;        // sixteens of a page: 1 to 8
    auto look_pages = [&](Lookup& u, int t0) {
      u.r = -1, u.page = -1;
      const int t = t0 + (lane >> 3);
      if (t >= my_tiles) return;
      const Segment g = segment_at(a_begin + t);
      const Span s = span_at(g.r);
      u.r = g.r, u.head = g.kvh, u.key = (s.lo / KT + g.first) * KT + 16 * sub;
      // a page of which no key is read is not fetched
      const int slot = u.key / p.page, first = slot * p.page;
      if (first <= s.hi && first + p.page > s.lo && slot < p.table_width) u.page = p.block_table[(size_t)g.r * p.table_width + slot];
    };
    auto look_scales = [&](Lookup& u) {
      const size_t where = (size_t)max(u.page, 0) * p.Hkv + (u.r < 0 ? 0 : u.head);
      u.ks = u.page >= 0 ? p.k_scale[where] : -1.f;
      u.vs = u.page >= 0 ? p.v_scale[where] : 1.f;
    };
    // a stage's barrier takes two arrivals: the copies asked for, the scales written
    const uint32_t page_bytes = (uint32_t)p.page * HD;
    auto copy = [&](int t, int s) {
      const bool there = (lane >> 3) == (t & 3) && now.page >= 0 && sub % per_page == 0;
      const int pages = __popc(__ballot_sync(0xffffffffu, there));
      const uint32_t full = smem_u32(&bars.full[s]);
      if (lane == 0) {
        if (pages > 0) mbar_arrive_expect_tx(full, 2 * pages * page_bytes);
        else mbar_arrive(full);
      }
      __syncwarp();
      if (there) {
        const uint32_t kdst = ring + s * S::STAGE + sub * 16 * HD;
        tma_load_4d(kdst, &k_map, full, 0, 0, now.head, now.page);
        tma_load_4d(kdst + S::OPERAND, &v_map, full, 0, 0, now.head, now.page);
      }
    };
    auto write_scales = [&](int t, int s) {
      if ((lane >> 3) == (t & 3)) bars.scales[s][sub] = make_float2(now.ks, fmaxf(log2f(now.vs), -100.f));
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars.full[s]));          // (after what the other lanes wrote)
    };
    // (a tile's copies take a third of a microsecond to ask for, their scales twice that to arrive: the first two tiles', then those)
    const int early = min(min(my_tiles, STAGES), 4);
    look_pages(now, 0);
    look_scales(now);
    for (int i = 0; i <= early; ++i) {
      if (i < early) copy(i, i);
      if (i > 0) write_scales(i - 1, i - 1);
    }
    look_pages(ahead, 4);
    int s = early % STAGES, par = early == STAGES ? 0 : 1, t = early;
    if (early == 4) look_scales(ahead);
    for (; t < my_tiles; ++t) {
      if ((t & 3) == 0) now = ahead, look_pages(ahead, t + 4);
      if ((t & 3) == 2 || (t == 3 && early == 3)) look_scales(ahead);
      bool ran_out;
      if (!mbar_wait_warp(smem_u32(&bars.empty[s]), par, aborted, ran_out)) {
        if (ran_out) gb_err::report(ERR_WAIT_EMPTY), *aborted = 1;
        break;
      }
      copy(t, s);
      write_scales(t, s);
      if (++s == STAGES) s = 0, par ^= 1;
    }
    if (*aborted && lane == 0 && t > 0) {
      // wind down: the copies in flight need microseconds to land; two milliseconds before the shared memory is given up
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {}
    }
  } else if (my_tiles > 0 && warp == 1) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t idesc_s = instr_desc(KT, N), idesc_o = instr_desc(KT, HD) | INSTR_B_MN_MAJOR;
    const uint64_t dk0 = smem_desc_rows<HD>(ring), dq0 = smem_desc_rows<HD>(q_at), dv0 = smem_desc_rows<HD>(ring + S::OPERAND),
                   dp0 = smem_desc_sw128(p_at);
    const bool leader = elect_one();
    bool ok = true, ran_out = false;
    int s = 0, par = 0, sp = 0;            // the stage of S^T and its phase, the stage of P V
    int seg_s = 0, left_s = 0, seg_o = 0, left_o = 0;      // segments begun (by S^T, by P V), tiles left of them
    int a_s = a_begin, a_o = a_begin;
    for (int t = 0; t <= my_tiles && ok; ++t) {
      if (t < my_tiles) {
        if (left_s == 0) {
          const Segment g = segment_at(a_s);
          left_s = g.count, a_s += g.count;
          ok = mbar_wait_warp(smem_u32(&bars.q_ready[seg_s & 1]), (seg_s >> 1) & 1, aborted, ran_out);
          ++seg_s;
        }
        if (ok) ok = mbar_wait_warp(smem_u32(&bars.full[s]), par, aborted, ran_out);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          const uint64_t dk = dk0 + (uint64_t)(s * (S::STAGE >> 4)), dq = dq0 + (uint64_t)(((seg_s - 1) & 1) * (S::Q_BYTES >> 4));
#pragma unroll
          for (int k = 0; k < HD / 32; ++k) mma_f8(tmem + (t & 1) * 32, dk + 2 * k, dq + 2 * k, idesc_s, k > 0);
          mma_commit(smem_u32(&bars.s_ready[t & 1]));
        }
        __syncwarp();
        --left_s;
        if (++s == STAGES) s = 0, par ^= 1;
      }
      if (t > 0) {
        const int u = t - 1;
        bool first = false;
        if (left_o == 0) {
          const Segment g = segment_at(a_o);
          left_o = g.count, a_o += g.count, first = true;
          // the results of the segment in front have been read
          if (seg_o > 0) ok = mbar_wait_warp(smem_u32(&bars.o_free), (seg_o - 1) & 1, aborted, ran_out);
          ++seg_o;
        }
        if (ok) ok = mbar_wait_warp(smem_u32(&bars.p_ready[u & 1]), (u >> 1) & 1, aborted, ran_out);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          const uint64_t dp = dp0 + (uint64_t)((u & 1) * (S::P_BYTES >> 4)), dv = dv0 + (uint64_t)(sp * (S::STAGE >> 4));
#pragma unroll
          for (int k = 0; k < KT / 32; ++k) mma_f8(tmem + O_COL, dp + 2 * k, dv + (uint64_t)(k * (32 * HD >> 4)), idesc_o, !first || k > 0);
          mma_commit(smem_u32(&bars.pv_done[u & 1]));
          mma_commit(smem_u32(&bars.empty[sp]));
        }
        __syncwarp();
        --left_o;
        if (++sp == STAGES) sp = 0;
      }
    }
    if (!ok) {
      if (ran_out && lane == 0) gb_err::report(ERR_WAIT_ACCUM);
      *aborted = 1;
    }
  } else if (my_tiles > 0) {
    // ---------------------------------------------------------------- scores and weights
    const int x = threadIdx.x - 64, quarter = warp & 3, sw = warp - 2;
    const int key_i = quarter * 32 + lane;                         // this thread's key of a tile
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    bool ok = true;
    auto wait = [&](uint64_t& bar, int phase) {
      if (ok && (!mbar_wait(smem_u32(&bar), phase & 1) || *aborted)) {
        if (!*aborted) gb_err::report(ERR_WAIT_ACCUM);
        ok = false, *aborted = 1;
      }
    };
    // the queries of a segment as codes: thread x has row x / (HD / 16), 16 channels
    uint4 raw[2];
    const int qrow = x / (HD / 16), qc = x % (HD / 16);
    auto ask_queries = [&](const Segment& g) {
      const Span s = span_at(g.r);
      const bool there = qrow < s.nrows && qrow < ROWS;
      const uint4* src = reinterpret_cast<const uint4*>(
          p.q + ((size_t)(s.q_begin + (there ? qrow / p.g : 0)) * p.Hq + g.kvh * p.g + (there ? qrow % p.g : 0)) * HD + 16 * qc);
      raw[0] = there ? src[0] : make_uint4(0u, 0u, 0u, 0u);
      raw[1] = there ? src[1] : make_uint4(0u, 0u, 0u, 0u);
    };
    auto put_queries = [&](int seg) {
      const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
      uint32_t hi[4], lo[4];
      const float unit = split_query<HD / 16>(w, 16.f, hi, lo);
      if (qrow < ROWS) {
        uint8_t* to = base + 2 * S::P_BYTES + (seg & 1) * S::Q_BYTES;
        *reinterpret_cast<uint4*>(to + swizzled<HD>(qrow, qc)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(to + swizzled<HD>(qrow + ROWS, qc)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (qc == 0) bars.factor[seg & 1][qrow] = unit * p.scale_log2;
      }
      fence_proxy_async();            // the tensor core reads them through the async proxy
      mbar_arrive(smem_u32(&bars.q_ready[seg & 1]));
    };
    // segments that other CTAs have a part of: the first and the last at most; merged at the end
    struct Shared {
      Segment g;
      int nrows, q_begin;
    } shared[2];
    int n_shared = 0, t = 0, s = 0, par = 0;
    // the queries of a segment are put while the one in front is at work, and asked for one segment earlier still
    Segment now = segment_at(a_begin), next, later;
    int a = a_begin;
    ask_queries(now);
    put_queries(0);
    sync_four();                      // the factors
    if (a + now.count < a_end) next = segment_at(a + now.count), ask_queries(next);
    for (int seg = 0; a < a_end; ++seg) {
      const Segment g = now;
      const Span w = span_at(g.r);
      bool asked = a + g.count < a_end;
      // per row: the reference, in powers of two, and the denominator, the sum of 2^(s - ref); of the keys up to the last change of references
      // the largest vs
      float ref[ROWS], l[ROWS], vtop = -200.f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) ref[r] = -INFINITY, l[r] = 0.f;

      for (int j = 0; j < g.count; ++j, ++t) {
        wait(bars.s_ready[t & 1], t >> 1);
        wait(bars.full[s], par);                   // (over already)
        tc_fence_after_sync();
        const float2 sc = bars.scales[s][key_i >> 4];
        const int key0 = (w.lo / KT + g.first + j) * KT, key = key0 + key_i;
        const bool readable = key >= w.lo && key <= w.hi && sc.x >= 0.f;
        // no mask for a tile that lies before the first row's position, inside the last row's window, on pages that are there
        const bool full = key0 + KT - 1 <= w.pos0 && (p.window <= 0 || key0 >= w.hi + 1 - p.window) && sc.x >= 0.f;
        float u[ROWS];                             // log2 of exp(s) * vs
        {
          uint32_t raw_s[N];
          tmem_load<N>(lane_addr + (t & 1) * 32, raw_s);
          tmem_ld_wait();
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            u[r] = fmaf(fmaf(__uint_as_float(raw_s[r + ROWS]), 0.0625f, __uint_as_float(raw_s[r])), bars.factor[seg & 1][r] * sc.x, sc.y);
        }
        if (!full) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const int pos = w.pos0 + r / p.g;
            if (!readable || key > pos || (p.window > 0 && key + p.window <= pos)) u[r] = -INFINITY;
          }
          // A value row that nobody reads is cleared: a weight of zero times a code that is no number would spoil a sum.
          if (!readable) {
            uint8_t* row = base + S::RING_AT + s * S::STAGE + S::OPERAND + key_i * HD;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) reinterpret_cast<uint4*>(row)[c] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        const float ev = readable ? sc.y : -200.f;
        bool more = false;
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < w.nrows) more = more || !(u[r] <= ref[r] + S::GROWTH);          // (a score that is no number stays one)
        // a key far above the reference (rare after a request's first tiles): everything is brought to it
        if (j == 0 || any_of_four(more)) {
          if (j > 0) {
            wait(bars.pv_done[(t - 1) & 1], (t - 1) >> 1);
            tc_fence_after_sync();
          }
          const float vt = redux_max(ev);
          if (lane == 0) bars.vtop[sw] = vt;
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            if (r < w.nrows) {
              const float top = redux_max(u[r]);
              if (lane == 0) bars.top[sw][r] = top;
            }
          sync_four();
          vtop = fmaxf(vtop, fmaxf(fmaxf(bars.vtop[0], bars.vtop[1]), fmaxf(bars.vtop[2], bars.vtop[3])));
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            if (r >= w.nrows) continue;
            const float top = fmaxf(ref[r], fmaxf(fmaxf(bars.top[0][r], bars.top[1][r]), fmaxf(bars.top[2][r], bars.top[3][r])));
            const float corr = ref[r] == -INFINITY ? 0.f : exp2_fast(ref[r] - top);
            if (j > 0 && ref[r] != -INFINITY) l[r] = times_power(l[r], ref[r] - top);
            ref[r] = top;
            if (x == r) bars.corr[r] = corr;
          }
          sync_four();               // (before the maxima's place is used again, too)
          if (quarter == 0 && j > 0) {             // the sums' rows lie in its lanes: r, r + ROWS, r + 2 ROWS
            const float corr = lane < S::PARTS * ROWS && lane % ROWS < w.nrows ? bars.corr[lane % ROWS] : 1.f;
#pragma unroll 1                           // (unrolled, registers of the whole tile's turn went to memory: 4 x 65,536 keys 100 us for 90)
            for (int h = 0; h < HD / 32; ++h) {
              uint32_t o[32];
              tmem_ld_32(lane_addr + O_COL + h * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
              tmem_st_32(lane_addr + O_COL + h * 32, o);
            }
            tmem_st_wait();
          }
        }
        if (t >= 2) wait(bars.pv_done[t & 1], (t - 2) >> 1);       // P's buffer is free
        // Weights times vs, in units of 2^(ref - UP), as codes; the denominator takes vs out again. Only where this key's vs is 2^-90 of another's may
        // its weight be too small a number for that, and count all the same: the denominator gets an exponential of its own.
        const bool far = sc.y < vtop - 90.f;
        if (far) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            if (r < w.nrows) l[r] += exp2_fast(u[r] - sc.y - (ref[r] == -INFINITY ? 0.f : ref[r]));
        }
        const float down = far ? 0.f : exp2_fast(-S::UP - sc.y);
        const uint32_t p_base = p_at + (t & 1) * S::P_BYTES + (key_i & 15), chunk = (uint32_t)key_i >> 4;
#pragma unroll
        for (int r = 0; r < ROWS; r += 2) {
          if (r >= w.nrows) break;
          const float wa = exp2_fast(u[r] + (S::UP - (ref[r] == -INFINITY ? 0.f : ref[r])));
          const float wb = exp2_fast(u[r + 1] + (S::UP - (ref[r + 1] == -INFINITY ? 0.f : ref[r + 1])));
          l[r] = fmaf(wa, down, l[r]), l[r + 1] = fmaf(wb, down, l[r + 1]);
          uint32_t code[S::PARTS];
          split<S::PARTS>(wa, wb, code);
          // row r of P: 128 bytes, its chunks of 16 swizzled
          const uint32_t a0 = p_base + r * 128 + ((chunk ^ (r & 7)) << 4), a1 = p_base + (r + 1) * 128 + ((chunk ^ ((r + 1) & 7)) << 4);
#pragma unroll
          for (int i = 0; i < S::PARTS; ++i) st_shared_u8(a0 + i * ROWS * 128, code[i]), st_shared_u8(a1 + i * ROWS * 128, code[i] >> 8);
        }
        fence_proxy_async();            // the tensor core reads weights and values through the async proxy
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&bars.p_ready[t & 1]));
        if (++s == STAGES) s = 0, par ^= 1;
        if (asked && (j == 1 || j + 1 == g.count)) {
          put_queries(seg + 1);
          asked = false;
          if (a + g.count + next.count < a_end) later = segment_at(a + g.count + next.count), ask_queries(later);
        }
      }
      // ---- the segment's results
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (r < w.nrows) {
          const float sum = gb::warp_sum(l[r]);
          if (lane == 0) bars.lsum[sw][r] = sum;
        }
      wait(bars.pv_done[(t - 1) & 1], (t - 1) >> 1);
      tc_fence_after_sync();
      sync_four();
      const bool whole = g.first == 0 && g.count == g.n;
      if (quarter == 0) {
        const int r = lane % ROWS;
        const bool mine = lane < w.nrows && ok;
        float mine_ref = -INFINITY;
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          if (i == r) mine_ref = ref[i];
        const float ll = (bars.lsum[0][r] + bars.lsum[1][r]) + (bars.lsum[2][r] + bars.lsum[3][r]);
        const float unit = exp2_fast(-S::UP), inv = ll > 0.f ? 1.0f / ll : ll == ll ? 0.f : ll;
        const float f = whole ? unit * inv : unit;
        __nv_bfloat16* const dst = p.out + ((size_t)(w.q_begin + r / p.g) * p.Hq + g.kvh * p.g + r % p.g) * HD;
        float* const part = partials + ((size_t)cta * 2 + (a == a_begin ? 0 : 1)) * (MAX_ROWS * RS) + r * RS;
        float* const own_part = reinterpret_cast<float*>(base + S::PARTS_AT) + (rank * ROWS + r) * S::RC;
        const uint32_t to = CLUSTER ? map_to_rank(smem_u32(own_part), 0) : 0;
#pragma unroll 1
        for (int h = 0; h < HD / 16; ++h) {
          uint32_t o[16];
          tmem_ld_16(lane_addr + O_COL + h * 16, o);
          tmem_ld_wait();
          float y[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float hi = __uint_as_float(o[c]);
            float lo = __shfl_sync(0xffffffffu, hi, (lane + ROWS) & 31);
            if (S::PARTS == 3) lo = fmaf(__shfl_sync(0xffffffffu, hi, (lane + 2 * ROWS) & 31), 0.03125f, lo);
            // (nothing seen: the sums mean nothing)
            y[c] = mine_ref == -INFINITY && ll == ll ? 0.f : fmaf(lo, 0.03125f, hi) * f;
          }
          if (CLUSTER && mine && !whole) {
#pragma unroll
            for (int c = 0; c < 16; c += 4) st_cluster_v4(to + (h * 16 + c) * 4, y[c], y[c + 1], y[c + 2], y[c + 3]);
          } else if (mine) {
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              if (whole) gb::store_pair(dst + h * 16 + c, y[c], y[c + 1]);
              else __stcg(reinterpret_cast<float2*>(part + h * 16 + c), make_float2(y[c], y[c + 1]));
            }
          }
        }
        if (CLUSTER && mine && !whole) {
          st_cluster_v4(to + HD * 4, mine_ref, ll, 0.f, 0.f);
        } else if (mine && !whole) {
          __stcg(reinterpret_cast<float2*>(part + HD), make_float2(mine_ref, ll));
        }
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&bars.o_free));
      }
      if (!whole) {
        const Shared y = {g, w.nrows, w.q_begin};
        if (n_shared == 0) shared[0] = y;
        else shared[1] = y;
        ++n_shared;
      }
      a += g.count;
      now = next, next = later;
    }
    // ---- segments of several CTAs: who counts the last arrival adds the parts up, in the CTAs' order
    if (CLUSTER) {
      __syncwarp();
      cluster_arrive_wait();           // (every thread of the cluster once, the others at the kernel's end; every wait in front of it is bounded)
      if (rank != 0) n_shared = 0;
    } else if (n_shared > 0) {
      sync_four();                     // the parts are written
    }
    int c0[2] = {0, 0}, c1[2] = {0, 0};
    bool behind[2] = {false, false};   // whether the first of them has another segment's end in front of its part
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (CLUSTER) c1[i] = (own_n + own_per - 1) / max(own_per, 1) - 1;
      if (CLUSTER || i >= n_shared) break;
      const Segment& g = shared[i].g;
      const int c = cost[g.r] * p.Hkv + g.kvh * (g.n + SEGMENT);
      c0[i] = c / stretch, c1[i] = (c + g.n - 1) / stretch;
      behind[i] = begins_at(c0[i]) < cum[g.r] * p.Hkv + g.kvh * g.n;
    }
    if (!CLUSTER && x < n_shared) {
      __threadfence();
      const Segment& g = x == 0 ? shared[0].g : shared[1].g;
      int* counter = counters + (size_t)g.r * p.Hkv + g.kvh;
      const bool last = atomicAdd(counter, 1) == (x == 0 ? c1[0] - c0[0] : c1[1] - c0[1]);
      if (last) *counter = 0;                        // as the next launch expects it
      bars.last[x] = last;
      __threadfence();
    }
    if (!CLUSTER && n_shared > 0) sync_four();
    constexpr int LANES = 128 / ROWS, PER = HD / LANES / 2;          // threads of a row, pairs of channels of a thread
    const int row = x / LANES, sub = x % LANES;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i >= n_shared || (!CLUSTER && !bars.last[i]) || row >= shared[i].nrows || !ok) continue;
      auto part_of = [&](int c) -> const float* {
        if (CLUSTER) return reinterpret_cast<const float*>(base + S::PARTS_AT) + (c * ROWS + row) * S::RC;
        return partials + ((size_t)c * 2 + (c == c0[i] && behind[i] ? 1 : 0)) * (MAX_ROWS * RS) + row * RS;
      };
      auto read2 = [&](const float* from) { return CLUSTER ? *reinterpret_cast<const float2*>(from) : __ldcg(reinterpret_cast<const float2*>(from)); };
      float top = -INFINITY, ll = 0.f;
      float2 v[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int c = c0[i]; c <= c1[i]; c += 4) {        // four parts' loads under way at once
        float2 ml[4], y[4][PER];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* part = part_of(min(c + k, c1[i]));
          ml[k] = read2(part + HD);
#pragma unroll
          for (int e = 0; e < PER; ++e) y[k][e] = read2(part + 2 * (sub + LANES * e));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c + k > c1[i]) break;
          const float top_new = fmaxf(top, ml[k].x);
          const float old = top == -INFINITY ? 0.f : exp2_fast(top - top_new), f = ml[k].x == -INFINITY ? 0.f : exp2_fast(ml[k].x - top_new);
          if (top != -INFINITY) ll = times_power(ll, top - top_new);
          ll += ml[k].x == -INFINITY ? (ml[k].y == ml[k].y ? 0.f : ml[k].y) : times_power(ml[k].y, ml[k].x - top_new);          // (a part without a key has nothing)
          top = top_new;
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            v[e].x = v[e].x * old + (f > 0.f ? f * y[k][e].x : 0.f);
            v[e].y = v[e].y * old + (f > 0.f ? f * y[k][e].y : 0.f);
          }
        }
      }
      const float inv = ll > 0.f ? 1.0f / ll : ll == ll ? 0.f : ll;
      const Segment& g = shared[i].g;
      __nv_bfloat16* const dst = p.out + ((size_t)(shared[i].q_begin + row / p.g) * p.Hq + g.kvh * p.g + row % p.g) * HD;
#pragma unroll
      for (int e = 0; e < PER; ++e) gb::store_pair(dst + 2 * (sub + LANES * e), v[e].x * inv, v[e].y * inv);
    }
  }
  if (CLUSTER && (my_tiles == 0 || warp < 2)) {
    __syncwarp();
    cluster_arrive_wait();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// ------------------------------------------------------------------ host side
constexpr int CLUSTER_TILES = 16;
constexpr int MAX_REQUESTS = 256;    // of one launch: their lengths lie in shared memory

template <int HD, int N, bool CLUSTER>
int launch(const Params& p, const CUtensorMap& km, const CUtensorMap& vm, long long tiles_most, int min_tiles, void* parts, void* counters,
           cudaStream_t stream) {
  using S = Shape<HD, N, CLUSTER>;
  auto kernel = attention_f8_decode_kernel<HD, N, CLUSTER>;
  constexpr int LENGTHS = (4 * MAX_REQUESTS + 3) * 4;
  static_assert(1024 + S::BYTES + LENGTHS + (int)sizeof(Bars) + 1024 <= 232448, "one CTA");
  static_assert(S::CTAS == 1 || 2 * (1024 + S::BYTES + LENGTHS + (int)sizeof(Bars) + 1024) <= 233472, "two CTAs an SM");
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 1024 + S::BYTES + LENGTHS);
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "attention_f8_decode: %s", cudaGetErrorString(e));
    configured.done();
  }
  const int room = tc_host::sm_count() * S::CTAS;
  const long long most = std::max(tiles_most / min_tiles + 1, (long long)p.R * p.Hkv);
  const size_t smem = 1024 + S::BYTES + (size_t)(4 * p.R + 3) * 4;
  const unsigned grid = CLUSTER ? (unsigned)(p.R * p.Hkv * min_tiles) : (unsigned)(most < room ? most : room);
  return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3(grid), dim3(THREADS), smem, stream, dim3(CLUSTER ? (unsigned)min_tiles : 1u), km, vm, p,
                                             min_tiles, (float*)parts, (int*)counters), "attention_f8_decode");
}

}  // namespace

// Bytes of the parts that CTAs leave to one another (no need to clear them). The counters are four bytes for each request and head, zero before the
// first launch; every launch leaves them zero.
GB_EXPORT long long gb_f8_attention_decode_part_bytes() { return (long long)tc_host::sm_count() * 2 * 2 * MAX_ROWS * (128 + 2) * 4; }

// The most rows (new tokens times heads of a group) of a request that the next entry takes, in groups of g heads; 0: it takes none.
GB_EXPORT int gb_f8_attention_decode_rows(int g) { return decode_rows(g); }

// Heads of 64 or 128, pages of 16, 32, 64 or 128 keys, up to sixteen query heads a group; for requests of up to decode_rows(g) rows (new tokens
// times heads of a group), the others are left.
GB_EXPORT int gb_f8_attention_decode(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale, const void* table,
                                     int table_width, const void* cu_q, const void* kv_lens, void* out, int R, long long pages, int Hq, int Hkv, int hd,
                                     float scale, int window, int page, int max_kv_len, void* parts, void* counters, void* stream) {
  if (R <= 0 || Hkv <= 0 || Hq % Hkv || (hd != 64 && hd != 128) || page < 16 || page > 128 || (page & (page - 1)) ||
      Hq / Hkv > MAX_ROWS || (uintptr_t)q % 16 || (uintptr_t)out % 4 ||
      (uintptr_t)k_pool % 16 || (uintptr_t)v_pool % 16)
    return gb::fail(GB_BAD_ARGUMENT, "attention_f8_decode: %d requests, heads %d / %d of %d, pages of %d", R, Hq, Hkv, hd, page);
  CUtensorMap km, vm;
  int rc = pool_map(k_pool, page, Hkv, pages, hd, &km);
  if (rc) return rc;
  rc = pool_map(v_pool, page, Hkv, pages, hd, &vm);
  if (rc) return rc;
  const int g = Hq / Hkv, reach = window > 0 && window + 2 * KT < max_kv_len ? window + 2 * KT : max_kv_len;
  const int min_tiles = 4;
  if (((long long)(reach + KT - 1) / KT + 4) * Hkv * (R < MAX_REQUESTS ? R : MAX_REQUESTS) > (1ll << 30))
    return gb::fail(GB_UNSUPPORTED, "attention_f8_decode: %d requests of %d positions", R, reach);
  for (int r0 = 0; r0 < R && rc == GB_OK; r0 += MAX_REQUESTS) {
    const int n = R - r0 < MAX_REQUESTS ? R - r0 : MAX_REQUESTS;
    const Params p{(const __nv_bfloat16*)q, (const float*)k_scale, (const float*)v_scale, (__nv_bfloat16*)out,
                   (const int32_t*)table + (size_t)r0 * table_width, (const int32_t*)cu_q + r0, (const int32_t*)kv_lens + r0, table_width, n, Hq,
                   Hkv, g, window, page, scale * 1.4426950408889634f};
    const int reach_tiles = (reach + KT - 1) / KT;
    const long long tiles = (long long)n * Hkv * (reach_tiles + 1);
    int* count = (int*)counters + (size_t)r0 * Hkv;
    const cudaStream_t st = (cudaStream_t)stream;
    // Few heads with little work: a cluster for each, which merges through shared memory and sums no lengths up: eight CTAs, or as many as let all
    // clusters run at once (the GPU holds 15 of eight, 22 of six, 33 of four, one CTA an SM; with three CTAs for 48 heads a third of them
    // waited: 19 us for 10.6 with two). Heads of 128, eight of them, us with and without clusters: 500 keys 7.6 / 11.8, 2,048 9.5 / 15.7, 8,192
    // 14.9 / 18.5, 16,384 22.0 / 23.8; 64 heads: 500 keys 9.5 / 12.8, 2,048 15.6 / 20.1, 4,096 22.5 / 25.6. Not where a CTA gets more
    // than CLUSTER_TILES tiles (22 of them: 27.2 / 27.0): requests of unequal length are not evened out here.
    const int heads = n * Hkv;
    int c = heads <= 15 ? 8 : heads <= 22 ? 6 : heads <= 33 ? 4 : heads <= tc_host::sm_count() / 2 ? 2 : heads <= tc_host::sm_count() ? 1 : 0;
    c = std::min(std::min(c, MAX_CLUSTER), reach_tiles);
    const bool cluster = c >= 1 && (reach_tiles + c - 1) / c <= CLUSTER_TILES;
    const auto go = [&](auto hd_c, auto n_c) {
      constexpr int HD = decltype(hd_c)::value, N = decltype(n_c)::value;
      return cluster ? launch<HD, N, true>(p, km, vm, tiles, c, parts, count, st) : launch<HD, N, false>(p, km, vm, tiles, min_tiles, parts, count, st);
    };
    using std::integral_constant;
    if (hd == 64) rc = g <= 8 ? go(integral_constant<int, 64>(), integral_constant<int, 16>()) : go(integral_constant<int, 64>(), integral_constant<int, 32>());
    else rc = g <= 8 ? go(integral_constant<int, 128>(), integral_constant<int, 16>()) : go(integral_constant<int, 128>(), integral_constant<int, 32>());
  }
  return rc;
}

GB_EXPORT int gb_f8_attention_decode_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_f8_attention_decode_set_error_sink(void* host_word) { return gb_err::set_sink((int*)host_word); }
