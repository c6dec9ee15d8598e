// Attention of prompt portions over pages of E4M3 codes with a scale per page and head, on the fifth-generation tensor cores.
//
//   s_j = (q . k8_j) * ks(page of j) * scale over keys [start, pos];  out = sum_j softmax(s)_j vs(page of j) v8_j
// (garuda/src/llama/mod.rs:793-818; the window garuda/src/cache/mod.rs:333-338; query head h reads key/value head h / g).
//
// Laid out as the bfloat16 kernel (attention_tcgen05.cu): 128 query rows a piece of work, tiles of 128 keys, persistent CTAs, S = Q K^T two
// tiles ahead of O += P V, two softmax groups of 128 threads with 64 keys of every tile each and an accumulator of their own,
// probabilities through tensor memory, a reference maximum that moves when it has been outgrown by 2^8. What the codes change:
//   * S is a product of codes as they lie (tcgen05.mma kind f8f6f4): a query row, scaled by a power of two to a largest of at most 448, is the
//     sum of two E4M3 rows (a bfloat16's eight bits are four and four; what is 2^-11 of the row's largest and below loses bits
//     that the sum does not see), so S = Qhi K^T + Qlo K^T at twice the rate of bfloat16: the same time, half of the keys' bytes.
//   * Values become halves (exactly: every E4M3 number is one) in shared memory, a conversion for two of them, by four warps of
//     their own: 128 keys of 128 channels are 256 conversions and 1,024 shared-memory accesses of 16 bytes a warp lane row, for 128 rows'
//     worth of products. (Splitting P into codes instead would cost the softmax warps, which set the pace, two instructions a score.)
//   * A page's ks goes into the factor of the exponent's multiply-add, its vs (as a power of two) into the constant; the denominator takes it
//     out again per sixteen keys. The accumulators are in units of the largest vs so far. P in halves: eleven bits.
//   warp 0      TMA: keys and values, a box a page, into rings of their own; looks up pages and scales four tiles at a time, two steps ahead
//   warp 1      one elected lane issues the products
//   warps 4-11  softmax
//   warps 12-15 the queries of the next piece as codes, the values of the next tile as halves (rows that no query reads as zeros)
// Registers are shared out by need (setmaxnreg). Every wait is bounded.
#include "attention_float8.cuh"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace {

using namespace tc;
using attn8::Params;

constexpr int QROWS = 128;          // query rows per CTA
constexpr int KT = 128;             // keys per tile
constexpr int GROUPS = 2;           // softmax groups: each walks its own half of every key tile
constexpr int GK = KT / GROUPS;     // keys per group and tile
constexpr int BLOCK_BYTES = 128 * 128;              // 128 values' rows of one block of 64 channels in halves
constexpr int TMEM_COLS = 512;
constexpr int S_BUFS = 2;                           // S buffers: the S products run this many tiles ahead
constexpr int O_COL0 = S_BUFS * KT;                 // behind the S buffers
constexpr int THREADS = 512;
constexpr float RESCALE_ABOVE = 8.f;                // in powers of two
constexpr float UP = 6.f;                           // probabilities are multiplied by 2^6: halves go to 65,504, and down to 2^-30 of the reference
constexpr int SLOTS = 16;                            // tiles' scales in flight
// registers a thread of the warpgroups: copies and products, softmax (two), conversions; 128 a thread at launch
constexpr int REGS_ISSUE = 56, REGS_SOFTMAX = 176, REGS_CONVERT = 104;
static_assert(REGS_ISSUE + 2 * REGS_SOFTMAX + REGS_CONVERT <= 4 * 128, "no more registers than at launch");

template <int HD>
struct Shape {
  static constexpr int BLOCKS = HD / 64;                              // blocks of 64 channels of values in halves
  static constexpr int Q_BYTES = 2 * QROWS * HD, CODE_BYTES = KT * HD, H_BYTES = BLOCKS * BLOCK_BYTES;
  static constexpr int K_STAGES = HD == 64 ? 4 : 3, V_STAGES = HD == 64 ? 4 : 2, H_STAGES = HD == 64 ? 3 : 2;
  static constexpr int K_AT = 2 * Q_BYTES, V_AT = K_AT + K_STAGES * CODE_BYTES, H_AT = V_AT + V_STAGES * CODE_BYTES;
  static constexpr int TILE_BYTES = H_AT + H_STAGES * H_BYTES;
  static constexpr int CH = HD / GROUPS;                              // channels that a group writes out in the merge
  static_assert(O_COL0 + GROUPS * HD <= TMEM_COLS && GK == 64, "tensor memory layout");
  static_assert(K_STAGES + 5 <= SLOTS, "a tile's scales outlive its keys");
};

// Barriers and the like, behind the tiles in dynamic shared memory.
struct Misc {
  uint64_t q_full[2], q_empty[2], k_full[6], k_empty[6], v_full[4], v_empty[4], h_full[3], h_empty[3];
  uint64_t s_ready[S_BUFS], p_ready[S_BUFS], o_ready;
  uint32_t tmem_base;
  int abort;
  float2 scales[SLOTS][8];              // a tile's ks of each sixteen keys (negative: no page there) and log2 of vs
  float factor[2][QROWS];               // per query row: 2^e * scale * log2(e)
  float2 ml[GROUPS][QROWS];             // the groups' reference maxima and denominators, for the merge
  float vref[GROUPS];
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// The largest of three in one instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Sums in 32 bits; E4M3 operands, or (the same bits) halves.
__device__ __forceinline__ constexpr uint32_t instr_desc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Rows of 128 bytes (or of 64) as TMA swizzles them, eight to a group.
template <int HD>
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t addr) {
  if (HD == 128) return smem_desc_sw128(addr);
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(512 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
}
// Byte offset of 16-byte chunk `c` of row `row` in such a tile.
template <int HD>
__device__ __forceinline__ uint32_t swizzled(int row, int c) {
  return HD == 128 ? (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}

// One piece of work: 128 query rows of one request and kv head.
struct Item {
  bool valid;
  int kvh, q_begin, tok0, nrows, pos0, lo, hi, tile_begin, n_tiles;
  const int32_t* table;
};

// Items are numbered request by request, the tiles of a request from its end (the longest first), the
// kv heads innermost. A CTA takes every gridDim.x-th item, so each gets long and short ones.
__device__ __forceinline__ Item decode_item(const Params& p, int q_tiles, int item) {
  Item w;
  const int per_req = q_tiles * p.Hkv;
  const int r = item / per_req, rem = item % per_req;
  const int qt = q_tiles - 1 - rem / p.Hkv;
  w.kvh = rem % p.Hkv;
  // The batch's lengths and block tables were copied in before the step's first kernel.
  w.q_begin = p.cu_q[r];
  const int q_len = p.cu_q[r + 1] - w.q_begin;
  const int tokens_per_tile = QROWS / p.g;
  w.tok0 = qt * tokens_per_tile;
  w.valid = q_len * p.g > attn8::decode_rows(p.g) && w.tok0 < q_len;      // else a decode request, or past its end
  const int kv_len = p.kv_lens[r];
  const int ntok = min(tokens_per_tile, q_len - w.tok0);
  w.nrows = ntok * p.g;
  w.pos0 = kv_len - q_len + w.tok0;                                 // position of the tile's first token
  w.lo = p.window > 0 ? max(0, w.pos0 + 1 - p.window) : 0;          // first key any row reads
  w.hi = w.pos0 + ntok - 1;                                         // last key any row reads
  w.tile_begin = w.lo / KT;
  w.n_tiles = w.valid ? w.hi / KT + 1 - w.tile_begin : 0;
  w.table = p.block_table + (size_t)r * p.table_width;
  return w;
}

// Walks this CTA's items tile by tile.
// The k-th item of this CTA: rounds of gridDim.x items, walked forth and back in turn, so that the
// CTA that got the longest item of one round gets the shortest of the next.
__device__ __forceinline__ int cta_item(int k) {
  const int g = (int)gridDim.x, b = (int)blockIdx.x;
  return k * g + ((k & 1) ? g - 1 - b : b);
}

struct Cursor {
  int item, total, step, q_tiles, round;
  int it;          // valid items before this one
  int j;           // tile within the item
  Item w;
  bool done;
  __device__ __forceinline__ void seek(const Params& p) {
    done = true;
    while ((long long)round * step < total) {       // a round may end before this CTA's place in it
      if (item < total) {
        w = decode_item(p, q_tiles, item);
        if (w.valid) { done = false; break; }
      }
      item = cta_item(++round);
    }
  }
  __device__ __forceinline__ void start(const Params& p, int q_tiles_, int total_) {
    round = 0, step = gridDim.x, total = total_, q_tiles = q_tiles_, it = 0, j = 0;
    item = cta_item(0);
    seek(p);
  }
  __device__ __forceinline__ void next_item(const Params& p) {
    item = cta_item(++round), ++it, j = 0;
    seek(p);
  }
};

// The same walk for the warp that issues the matrix products: it needs nothing of an item but its
// number of tiles, and everything it executes delays the tensor cores. Its lanes decode 32 items at
// a time, one each; the walk then only shuffles the counts out.
struct TileWalk {
  int base;        // this CTA's items before the batch
  int my_n;        // tiles of this lane's item of the batch (0: none, or not a valid item)
  int lane_i;      // the current item's lane
  int n, j;        // the current item's tiles, the current tile
  int it;          // valid items before the current one
  bool done;
  __device__ __forceinline__ void load(const Params& p, int q_tiles, int total) {
    const int k = base + (int)(threadIdx.x & 31);
    const long long item = (long long)k * gridDim.x < total ? cta_item(k) : total;
    my_n = item < total ? decode_item(p, q_tiles, (int)item).n_tiles : 0;
  }
  __device__ __forceinline__ void seek(const Params& p, int q_tiles, int total) {
    for (;;) {
      // the next lane of the batch with tiles, if any
      const unsigned have = __ballot_sync(0xffffffffu, my_n > 0) & (0xffffffffu << lane_i);
      if (lane_i < 32 && have != 0) {
        lane_i = __ffs(have) - 1;
        n = __shfl_sync(0xffffffffu, my_n, lane_i);
        return;
      }
      base += 32;
      lane_i = 0;
      if ((long long)base * gridDim.x >= total) {
        done = true;
        return;
      }
      load(p, q_tiles, total);
    }
  }
  __device__ __forceinline__ void start(const Params& p, int q_tiles, int total) {
    base = 0, lane_i = 0, j = 0, it = 0, n = 0, done = false;
    load(p, q_tiles, total);
    seek(p, q_tiles, total);
  }
  __device__ __forceinline__ void next_tile(const Params& p, int q_tiles, int total) {
    if (++j >= n) {
      j = 0, ++it, ++lane_i;
      if (lane_i >= 32) lane_i = 32;
      seek(p, q_tiles, total);
    }
  }
};

// A persistent kernel: one CTA per SM takes items until none are left, keeping its tensor memory and
// barriers, so that the queries and first keys of the next item arrive, and its first S products
// run, while the last tiles of the one before are in the softmax.
template <int HD>
__global__ void __launch_bounds__(THREADS, 1)
attention_f8_tile_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Params p, const int q_tiles,
                         const int total_items) {
  using S = Shape<HD>;
  constexpr int K_STAGES = S::K_STAGES, V_STAGES = S::V_STAGES, H_STAGES = S::H_STAGES, BLOCKS = S::BLOCKS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Misc& mc = *reinterpret_cast<Misc*>(smem_raw + S::TILE_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t q_s = smem_u32(smem_raw);                         // two buffers: the rows' codes, then what they leave
  const uint32_t k_s = q_s + S::K_AT, v_s = q_s + S::V_AT, h_s = q_s + S::H_AT;
  if ((q_s & 1023u) != 0) {                                        // the swizzle needs it; never seen
    if (threadIdx.x == 0) gb_err::report(ERR_WAIT_DRAIN);
    return;
  }

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&mc.q_full[b]), 128);
      mbar_init(smem_u32(&mc.q_empty[b]), 1);
    }
    for (int b = 0; b < S_BUFS; ++b) {
      mbar_init(smem_u32(&mc.s_ready[b]), 1);
      mbar_init(smem_u32(&mc.p_ready[b]), GROUPS * 128);
    }
    for (int s = 0; s < K_STAGES; ++s) {
      mbar_init(smem_u32(&mc.k_full[s]), 1);
      mbar_init(smem_u32(&mc.k_empty[s]), 1);
    }
    for (int s = 0; s < V_STAGES; ++s) {
      mbar_init(smem_u32(&mc.v_full[s]), 1);
      mbar_init(smem_u32(&mc.v_empty[s]), 128);
    }
    for (int s = 0; s < H_STAGES; ++s) {
      mbar_init(smem_u32(&mc.h_full[s]), 128);
      mbar_init(smem_u32(&mc.h_empty[s]), 1);
    }
    mbar_init(smem_u32(&mc.o_ready), 1);
    mc.abort = 0;
    fence_barrier_init();
    fence_proxy_async();
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
  gb::pdl_wait();      // queries and this step's keys and values come from the kernel in front

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA
      // Lane i looks up sixteen keys: block i % 8 of tile i / 8 of four, over the items' borders; `ahead` holds the next four tiles.
      struct Lookup {
        int kvh, page;
        float ks, vs;
      } now{}, ahead{};
      const int sub = lane & 7, per_page = p.page >> 4;        // sixteens of a page: 1 to 8
      const uint32_t page_bytes = (uint32_t)p.page * HD;
      Cursor look;                  // the tile that is looked up next
      look.start(p, q_tiles, total_items);
      auto look_pages = [&](Lookup& u) {
        u.page = -1;
#pragma unroll 1
        for (int i = 0; i < 4 && !look.done; ++i) {
          if ((lane >> 3) == i) {
            const Item& w = look.w;
            u.kvh = w.kvh;
            // a page of which no key is read is not fetched
            const int key = (w.tile_begin + look.j) * KT + 16 * sub, slot = key / p.page, first = slot * p.page;
            if (first <= w.hi && first + p.page > w.lo && slot < p.table_width) u.page = w.table[slot];
          }
          if (++look.j >= look.w.n_tiles) look.next_item(p);
        }
      };
      auto look_scales = [&](Lookup& u) {
        const size_t where = (size_t)max(u.page, 0) * p.Hkv + u.kvh;
        u.ks = u.page >= 0 ? p.k_scale[where] : -1.f;
        u.vs = u.page >= 0 ? p.v_scale[where] : 1.f;
      };
      look_pages(now);
      look_scales(now);
      int gt = 0, ks = 0, kpar = 1, vs = 0, vpar = 1;       // tiles so far; the stages to fill and the phases of their "empty" barriers
      bool ok = true, ran_out;
      Cursor c;
      for (c.start(p, q_tiles, total_items); !c.done && ok; c.next_item(p)) {
        for (int j = 0; j < c.w.n_tiles && ok; ++j, ++gt) {
          if ((gt & 3) == 0) {
            if (gt > 0) now = ahead;
            look_pages(ahead);
          }
          if ((gt & 3) == 2) look_scales(ahead);
          const bool mine = (lane >> 3) == (gt & 3), there = mine && now.page >= 0 && sub % per_page == 0;
          const int pages = __popc(__ballot_sync(0xffffffffu, there));
          if (!(ok = mbar_wait_warp(smem_u32(&mc.k_empty[ks]), kpar, abort_s, ran_out))) break;
          if (mine) mc.scales[gt % SLOTS][sub] = make_float2(now.ks, log2f(now.vs));
          __syncwarp();
          if (lane == 0) {           // (after what the other lanes wrote)
            if (pages == 0) mbar_arrive(smem_u32(&mc.k_full[ks]));
            else mbar_arrive_expect_tx(smem_u32(&mc.k_full[ks]), pages * page_bytes);
          }
          __syncwarp();
          if (there) tma_load_4d(k_s + ks * S::CODE_BYTES + sub * 16 * HD, &k_map, smem_u32(&mc.k_full[ks]), 0, 0, now.kvh, now.page);
          if (++ks == K_STAGES) ks = 0, kpar ^= 1;
          if (!(ok = mbar_wait_warp(smem_u32(&mc.v_empty[vs]), vpar, abort_s, ran_out))) break;
          if (lane == 0) {
            if (pages == 0) mbar_arrive(smem_u32(&mc.v_full[vs]));
            else mbar_arrive_expect_tx(smem_u32(&mc.v_full[vs]), pages * page_bytes);
          }
          __syncwarp();
          if (there) tma_load_4d(v_s + vs * S::CODE_BYTES + sub * 16 * HD, &v_map, smem_u32(&mc.v_full[vs]), 0, 0, now.kvh, now.page);
          if (++vs == V_STAGES) vs = 0, vpar ^= 1;
        }
      }
      if (!ok) {
        if (ran_out) gb_err::report(ERR_WAIT_EMPTY);
        *abort_s = 1;
      }
      if (*abort_s && lane == 0) {
        // wind down: the copies in flight need microseconds to land; two milliseconds before the shared memory is given up
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {}
      }
    } else if (warp == 1) {
      // -------------------------------------------------------------------- MMA issuer
      // The S products run two tiles ahead of the P V products, across the items' borders. After a tile's softmax its P V goes first: it
      // reads the probabilities from the S buffer that the S product two tiles ahead then overwrites (products run in the order of
      // their issue).
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = instr_desc(QROWS, KT), idesc_o = instr_desc(QROWS, HD) | INSTR_B_MN_MAJOR;
      const uint64_t dq0 = smem_desc_rows<HD>(q_s), dk0 = smem_desc_rows<HD>(k_s), dv0 = smem_desc_sw128_mn(h_s, BLOCKS > 1 ? BLOCK_BYTES : 16);
      bool ok = true;
      TileWalk ws, wp;               // the S products' tile, the P V products' tile
      ws.start(p, q_tiles, total_items);
      wp = ws;
      int k_stage = 0, k_par = 0;                    // key stage (and its phase) of the S tile
      int h_stage = 0, h_par = 0;                    // value stage of the P V tile
      int s_buf = 0;                                 // S buffer of the S tile
      int p_buf = 0, p_par = 0;                      // buffer of the P V tile and its phase
      auto issue_s = [&]() {      // S = (Qhi + Qlo) K^T of the S tile into S buffer s_buf (both groups' columns)
        const int qb = ws.it & 1;
        if (ws.j == 0 && !mbar_wait(smem_u32(&mc.q_full[qb]), (ws.it >> 1) & 1)) ok = false;
        if (ok && !mbar_wait(smem_u32(&mc.k_full[k_stage]), k_par)) ok = false;
        if (!ok) {
          if (lane == 0) gb_err::report(ERR_WAIT_FULL);
          return;
        }
        tc_fence_after_sync();
        if (leader) {
          const uint64_t dq = dq0 + (uint64_t)(qb * (S::Q_BYTES >> 4)), dk = dk0 + (uint64_t)(k_stage * (S::CODE_BYTES >> 4));
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < HD / 32; ++k)
              mma_f8(tmem_base + s_buf * KT, dq + (uint64_t)(part * (QROWS * HD >> 4) + 2 * k), dk + 2 * k, idesc_s, part > 0 || k > 0);
          mma_commit(smem_u32(&mc.s_ready[s_buf]));      // the softmax warps pass it on to the keys' and the queries' "empty" barriers
        }
        __syncwarp();
        if (++k_stage == K_STAGES) k_stage = 0, k_par ^= 1;
        if (++s_buf == S_BUFS) s_buf = 0;
        ws.next_tile(p, q_tiles, total_items);
      };
#pragma unroll 1
      for (int b = 0; b < S_BUFS; ++b)
        if (ok && !ws.done) issue_s();
      while (ok && !wp.done) {
        if (*abort_s) break;
        if (ok && !mbar_wait(smem_u32(&mc.h_full[h_stage]), h_par)) {
          if (lane == 0) gb_err::report(ERR_WAIT_FULL);
          ok = false;
        }
        if (ok && !mbar_wait(smem_u32(&mc.p_ready[p_buf]), p_par)) {
          if (lane == 0) gb_err::report(ERR_WAIT_ACCUM);
          ok = false;
        }
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
#pragma unroll
          for (int g = 0; g < GROUPS; ++g)
            mma_bf16_ts<GK / 16>(tmem_base + O_COL0 + g * HD, tmem_base + p_buf * KT + g * GK,
                                 dv0 + (uint64_t)(h_stage * (S::H_BYTES >> 4) + g * (GK * 128 >> 4)), idesc_o, 16 * 128 >> 4, wp.j > 0);
          mma_commit(smem_u32(&mc.o_ready));             // the softmax warps pass it on to the values' "empty" barrier
        }
        __syncwarp();
        // both groups have read this S buffer in full, and the products above read their P from it
        // before the next one writes: the S product two tiles ahead takes the buffer over
        if (!ws.done) issue_s();
        if (!ok) break;
        if (++h_stage == H_STAGES) h_stage = 0, h_par ^= 1;
        if (++p_buf == S_BUFS) p_buf = 0, p_par ^= 1;
        wp.next_tile(p, q_tiles, total_items);
      }
      if (!ok) *abort_s = 1;
    }
  } else if (warp >= 12) {
    // -------------------------------------------------------------------- conversions
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONVERT));
    const int x = threadIdx.x - 384;             // a query row, a key
    bool ok = true;
    int gt = 0, vs = 0, vpar = 0, hs = 0, hpar = 1;
    // the queries of an item: this thread's row
    auto put_queries = [&](const Cursor& c) {
      const Item& w = c.w;
      const int qb = c.it & 1;
      if (c.it >= 2 && ok && (!mbar_wait(smem_u32(&mc.q_empty[qb]), ((c.it >> 1) & 1) ^ 1) || *abort_s)) {
        if (!*abort_s) gb_err::report(ERR_WAIT_EMPTY);
        ok = false, *abort_s = 1;
      }
      if (!ok) return;
      const bool there = x < w.nrows;
      const uint4* src = reinterpret_cast<const uint4*>(
          p.q + ((size_t)(w.q_begin + w.tok0 + (there ? x / p.g : 0)) * p.Hq + w.kvh * p.g + (there ? x % p.g : 0)) * HD);
      // (read twice, the second time from L1, rather than kept in 64 registers)
      float largest = 0.f;
#pragma unroll 4
      for (int i = 0; i < HD / 8; ++i) {
        const uint4 two = there ? src[i] : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t u[4] = {two.x, two.y, two.z, two.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) largest = max3(largest, fabsf(__uint_as_float(u[e] << 16)), fabsf(__uint_as_float(u[e] & 0xFFFF0000u)));
      }
      const int e2 = f8::scale_exponent(largest);
      const float inv = f8::power_of_two(-e2);
      uint8_t* to = smem_raw + qb * S::Q_BYTES;
#pragma unroll 2
      for (int i = 0; i < HD / 16; ++i) {
        const uint4 r0 = there ? src[2 * i] : make_uint4(0u, 0u, 0u, 0u), r1 = there ? src[2 * i + 1] : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t u[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = __uint_as_float(u[2 * e] << 16) * inv, b = __uint_as_float(u[2 * e] & 0xFFFF0000u) * inv;
          const float d = __uint_as_float(u[2 * e + 1] << 16) * inv, f = __uint_as_float(u[2 * e + 1] & 0xFFFF0000u) * inv;
          hi[e] = f8::encode4(a, b, d, f);
          const float4 back = f8::decode4(hi[e]);
          lo[e] = f8::encode4(a - back.x, b - back.y, d - back.z, f - back.w);
        }
        *reinterpret_cast<uint4*>(to + swizzled<HD>(x, i)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(to + QROWS * HD + swizzled<HD>(x, i)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      mc.factor[qb][x] = f8::power_of_two(e2) * p.scale_log2;
      fence_proxy_async();              // the tensor core reads them through the async proxy
      mbar_arrive(smem_u32(&mc.q_full[qb]));
    };
    Cursor c, next;
    c.start(p, q_tiles, total_items);
    next = c;
    if (!c.done) {
      put_queries(next);
      next.next_item(p);
    }
    for (; !c.done && ok; c.next_item(p)) {
      const Item& w = c.w;
      bool asked = !next.done;
      for (int j = 0; j < w.n_tiles && ok; ++j, ++gt) {
        if (!mbar_wait(smem_u32(&mc.v_full[vs]), vpar) || (ok && !mbar_wait(smem_u32(&mc.h_empty[hs]), hpar)) || *abort_s) {
          if (!*abort_s) gb_err::report(ERR_WAIT_FULL);
          ok = false, *abort_s = 1;
          break;
        }
        // this thread's key: its row of values, or zeros where no query may read it (a page that was not fetched, the unwritten end of the last
        // page: a probability of zero times a code that is no number would spoil a sum)
        const int key = (w.tile_begin + j) * KT + x;
        const bool readable = key >= w.lo && key <= w.hi && mc.scales[gt % SLOTS][x >> 4].x >= 0.f;
        const uint8_t* from = smem_raw + S::V_AT + vs * S::CODE_BYTES;
        uint8_t* to = smem_raw + S::H_AT + hs * S::H_BYTES;
        uint4 code[HD / 16];
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) code[i] = *reinterpret_cast<const uint4*>(from + swizzled<HD>(x, i));
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {          // sixteen channels: two chunks of halves
          const uint32_t u[4] = {readable ? code[i].x : 0u, readable ? code[i].y : 0u, readable ? code[i].z : 0u, readable ? code[i].w : 0u};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) h[2 * e] = f8::decode2_f16(u[e] & 0xFFFFu), h[2 * e + 1] = f8::decode2_f16(u[e] >> 16);
          uint8_t* block = to + (i >> 2) * BLOCK_BYTES;
          *reinterpret_cast<uint4*>(block + swizzled<128>(x, 2 * (i & 3))) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(block + swizzled<128>(x, 2 * (i & 3) + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        mbar_arrive(smem_u32(&mc.v_empty[vs]));
        fence_proxy_async();            // the tensor core reads them through the async proxy
        mbar_arrive(smem_u32(&mc.h_full[hs]));
        if (++vs == V_STAGES) vs = 0, vpar ^= 1;
        if (++hs == H_STAGES) hs = 0, hpar ^= 1;
        if (asked && (j == 1 || j + 1 == w.n_tiles)) {
          put_queries(next);
          next.next_item(p);
          asked = false;
        }
      }
    }
  } else {
    // -------------------------------------------------------------------- softmax warps
    // Group g takes keys [g * 64, g * 64 + 64) of every tile: an attention stream of its own
    // (reference maximum, denominator, accumulator), merged with the other group's at the end.
    // Two groups put two warps on every scheduler, so that one computes while the other waits
    // for tensor memory.
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int grp = (warp - 4) >> 2;
    const int quarter = warp & 3;                        // the TMEM lanes this warp may read
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_mine = lane_addr + O_COL0 + grp * HD;
    bool ok = true;       // false: this thread only keeps the others company at the barriers
    int gt = 0;           // tiles so far, over all items
    int sb = 0, sph = 0;          // the current tile's S buffer and the phase of its barriers
    int kstage = 0;               // the current tile's stage of keys
    int kpar = 0;
    int hprev = 0, hstage = 0;    // the values' stages of the tile before and of the current one
    const bool passes_on = threadIdx.x == 128;     // one thread tells the TMA warp what the tensor core has finished with
    Cursor c;
    for (c.start(p, q_tiles, total_items); !c.done; c.next_item(p)) {
      const Item& w = c.w;
      const int row_pos = row < w.nrows ? w.pos0 + row / p.g : -1;       // no key is valid for a padding row
      const int row_start = (row < w.nrows && p.window > 0) ? max(0, row_pos + 1 - p.window) : 0;
      float m = -INFINITY, l = 0.f;      // m: the reference maximum, in powers of two
      float vref = -200.f;               // log2 of the vs in whose units the sums are
      float factor = 0.f;

      // waits until the P V products of the tile counted t have ended
      auto wait_o = [&](int t) {
        if (!mbar_wait(smem_u32(&mc.o_ready), t & 1)) {
          if (lane == 0) gb_err::report(ERR_WAIT_ACCUM);
          ok = false;
          *abort_s = 1;
        }
        tc_fence_after_sync();
      };

      for (int j = 0; j < w.n_tiles && ok; ++j, ++gt) {
        if (*abort_s) { ok = false; break; }
        if (!mbar_wait(smem_u32(&mc.s_ready[sb]), sph)) {
          if (lane == 0) gb_err::report(ERR_WAIT_ACCUM);
          ok = false;
          *abort_s = 1;
          break;
        }
        mbar_wait(smem_u32(&mc.k_full[kstage]), kpar);        // (over already: the scales were written before it)
        tc_fence_after_sync();
        const uint32_t s_addr = lane_addr + sb * KT + grp * GK;
        // the row's 64 scores of this group, one wait for the two loads
        uint32_t sv[GK / 32][32];
#pragma unroll
        for (int h = 0; h < GK / 32; ++h) tmem_ld_32(s_addr + h * 32, sv[h]);
        if (j == 0) factor = mc.factor[c.it & 1][row];
        float f[4], ev[4];            // of each sixteen keys: the scores' factor, log2 of vs
        bool pages = true;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float2 two = mc.scales[gt % SLOTS][grp * 4 + b];
          f[b] = two.x * factor, ev[b] = two.x >= 0.f ? two.y : -200.f;
          pages = pages && two.x >= 0.f;
        }
        const int hcur = hstage;
        if (++hstage == H_STAGES) hstage = 0;
        const int tile_key0 = (w.tile_begin + j) * KT;
        tmem_ld_wait();
        if (passes_on) {      // S of this tile is complete: its keys have been read, and after an item's last tile its queries
          mbar_arrive(smem_u32(&mc.k_empty[kstage]));
          if (j == w.n_tiles - 1) mbar_arrive(smem_u32(&mc.q_empty[c.it & 1]));
        }
        if (++kstage == K_STAGES) kstage = 0, kpar ^= 1;
        auto sc = [&](int ch) -> float& { return reinterpret_cast<float&>(sv[ch >> 5][ch & 31]); };
        const int key0 = tile_key0 + grp * GK;
        // the keys need no mask if they lie wholly before the first row's position and inside the
        // last row's window
        const bool full = pages && key0 + GK - 1 <= w.pos0 && (p.window <= 0 || key0 >= w.hi + 1 - p.window);
        if (!full) {
#pragma unroll
          for (int ch = 0; ch < GK; ++ch)
            if (!(key0 + ch >= row_start && key0 + ch <= row_pos && f[ch >> 4] >= 0.f)) sc(ch) = -INFINITY;
          // (a factor must not turn a masked score's sign)
#pragma unroll
          for (int b = 0; b < 4; ++b) f[b] = fmaxf(f[b], 0x1p-126f);
        }
        // the maximum of each sixteen keys' raw products, times their factor
        float m_new = m;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float mx = max3(sc(16 * b), sc(16 * b + 1), sc(16 * b + 2));
#pragma unroll
          for (int ch = 3; ch < 15; ch += 2) mx = max3(mx, sc(16 * b + ch), sc(16 * b + ch + 1));
          mx = fmaxf(mx, sc(16 * b + 15));
          m_new = fmaxf(m_new, mx * f[b]);
        }
        const float ev_top = fmaxf(fmaxf(ev[0], ev[1]), fmaxf(ev[2], ev[3]));
        // The reference maximum moves only if some row of the warp has outgrown it by more than
        // 2^8; then the warp rescales what it has accumulated (the loads and stores of tensor
        // memory are the whole warp's). A row that has seen no valid key yet has nothing to rescale.
        const bool grown = (m != -INFINITY && m_new - m > RESCALE_ABOVE) || ev_top > vref;
        bool waited = false;
        if (j > 0 && __any_sync(0xffffffffu, grown)) {
          wait_o(gt - 1);
          waited = true;
          if (!ok) break;
          const float own = m == -INFINITY ? 1.f : fast_exp2(m - m_new);
          const float v_new = fmaxf(vref, ev_top), corr = own * fast_exp2(vref - v_new);
          vref = v_new;
#pragma unroll
          for (int h = 0; h < HD / 32; ++h) {
            uint32_t v[32];
            tmem_ld_32(o_mine + h * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int ch = 0; ch < 32; ++ch) v[ch] = __float_as_uint(__uint_as_float(v[ch]) * corr);
            tmem_st_32(o_mine + h * 32, v);
          }
          l *= own;
          m = m_new;
        } else {
          if (m == -INFINITY) m = m_new;
          vref = fmaxf(vref, ev_top);          // (j > 0: it is the larger one already)
        }
        const float neg_m = m == -INFINITY ? 0.f : -m;       // nothing valid yet: avoid inf - inf
        // All exponentials first, in place (the unit that computes them takes a warp's instruction
        // every eight cycles; the multiply-adds in front fit in between), then sums and packing.
        // (2^-100 of the largest vs is nothing; and where nothing is read the probabilities are zeros.)
        float up[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) up[b] = UP + fminf(fmaxf(ev[b] - vref, -100.f), 0.f);
#pragma unroll
        for (int ch = 0; ch < GK; ++ch) sc(ch) = fast_exp2(fmaf(sc(ch), f[ch >> 4], neg_m + up[ch >> 4]));   // exp2(-inf) = 0 for masked keys
        uint32_t pk[GK / 2];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float ls[2] = {0.f, 0.f};
#pragma unroll
          for (int ch = 16 * b; ch < 16 * b + 16; ch += 2) {
            ls[(ch >> 1) & 1] += sc(ch) + sc(ch + 1);
            pk[ch >> 1] = pack_f16(sc(ch), sc(ch + 1));
          }
          l = fmaf(ls[0] + ls[1], fast_exp2(-up[b]), l);          // without vs
        }
        tmem_st(s_addr, pk);            // over the first half of the scores just read
        tmem_st_wait();
        if (j > 0 && !waited) wait_o(gt - 1);      // every phase of the barrier is seen, in order
        tc_fence_before_sync();         // this thread's accesses to tensor memory are over
        mbar_arrive(smem_u32(&mc.p_ready[sb]));
        if (passes_on && j > 0) mbar_arrive(smem_u32(&mc.h_empty[hprev]));      // the tile before: its P V has ended
        hprev = hcur;
        if (++sb == S_BUFS) sb = 0, sph ^= 1;
      }
      if (ok && w.n_tiles > 0) {
        wait_o(gt - 1);
        if (passes_on && ok) mbar_arrive(smem_u32(&mc.h_empty[hprev]));
      }
      // ---- merge the groups: each writes its share of the channels, summed over all accumulators
      mc.ml[grp][row] = make_float2(m, l);
      if (row == 0) mc.vref[grp] = vref;
      tc_fence_before_sync();
      asm volatile("bar.sync 1, %0;" ::"n"(GROUPS * 128) : "memory");
      tc_fence_after_sync();
      if (ok && !*abort_s) {
        float a[GROUPS];
        float mt = -INFINITY, lt = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) mt = fmaxf(mt, mc.ml[g][row].x);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const float2 x = mc.ml[g][row];
          const float own = x.x == -INFINITY ? 0.f : fast_exp2(x.x - mt);
          lt += own > 0.f || x.y != x.y ? x.y * own : 0.f;        // (a score that is no number stays one)
          a[g] = own * fast_exp2(mc.vref[g] - UP);
        }
        const float inv = lt > 0.f ? 1.0f / lt : lt == lt ? 0.f : lt;
        __nv_bfloat16* dst = p.out + ((size_t)(w.q_begin + w.tok0 + row / p.g) * p.Hq + w.kvh * p.g + row % p.g) * HD + grp * S::CH;
#pragma unroll
        for (int h = 0; h < S::CH / 16; ++h) {
          float t[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) t[e] = lt == lt ? 0.f : lt;
#pragma unroll
          for (int g = 0; g < GROUPS; g += 2) {      // two accumulators at a time (registers)
            uint32_t v[2][16];
            tmem_ld_16(lane_addr + O_COL0 + g * HD + grp * S::CH + h * 16, v[0]);
            tmem_ld_16(lane_addr + O_COL0 + (g + 1) * HD + grp * S::CH + h * 16, v[1]);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) {      // a stream without a valid key has an accumulator that means nothing
              t[e] += a[g] > 0.f ? __uint_as_float(v[0][e]) * (a[g] * inv) : 0.f;
              t[e] += a[g + 1] > 0.f ? __uint_as_float(v[1][e]) * (a[g + 1] * inv) : 0.f;
            }
          }
          if (row < w.nrows) {
            uint4 w0, w1;
            w0.x = pack_bf16(t[0], t[1]), w0.y = pack_bf16(t[2], t[3]), w0.z = pack_bf16(t[4], t[5]), w0.w = pack_bf16(t[6], t[7]);
            w1.x = pack_bf16(t[8], t[9]), w1.y = pack_bf16(t[10], t[11]), w1.z = pack_bf16(t[12], t[13]), w1.w = pack_bf16(t[14], t[15]);
            *reinterpret_cast<uint4*>(dst + h * 16) = w0;
            *reinterpret_cast<uint4*>(dst + h * 16 + 8) = w1;
          }
        }
      }
      // The next item's first P V overwrites the accumulators; it is issued only after all groups
      // have arrived for that tile, that is after all are through here. A
      // group must not write the next item's values while another still reads these.
      asm volatile("bar.sync 1, %0;" ::"n"(GROUPS * 128) : "memory");
      tc_fence_before_sync();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// ------------------------------------------------------------------ host side
struct MapKey {
  const void* ptr;
  long long page, heads, pages;
  int hd;
  bool operator==(const MapKey& o) const { return ptr == o.ptr && page == o.page && heads == o.heads && pages == o.pages && hd == o.hd; }
};
struct MapKeyHash {
  size_t operator()(const MapKey& k) const {
    return std::hash<const void*>()(k.ptr) ^ (std::hash<long long>()(k.page) * 31) ^ (std::hash<long long>()(k.heads) * 131) ^
           (std::hash<long long>()(k.pages) * 521) ^ (size_t)k.hd * 7919;
  }
};

// Pools [pages][heads][page][hd] of bytes through boxes [1][1][page][hd], swizzled over the rows' width.
int pool_map(const void* ptr, int page, int heads, long long pages, int hd, CUtensorMap* out) {
  static std::mutex mu;
  static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
  const MapKey key{ptr, page, heads, pages, hd};
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(key);
  if (it != cache.end()) {
    *out = it->second;
    return GB_OK;
  }
  tc_host::EncodeTiledFn fn = tc_host::encode_fn();
  if (!fn) return gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)page, (cuuint64_t)heads, (cuuint64_t)pages};
  cuuint64_t strides[3] = {(cuuint64_t)hd, (cuuint64_t)hd * page, (cuuint64_t)hd * page * heads};
  cuuint32_t box[4] = {(cuuint32_t)hd, (cuuint32_t)page, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUtensorMap m;
  const CUresult r = fn(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled failed with code %d for a pool of codes", (int)r);
  if (cache.size() >= 1024) cache.clear();
  cache.emplace(key, m);
  *out = m;
  return GB_OK;
}

template <int HD>
int launch(const Params& p, const CUtensorMap& km, const CUtensorMap& vm, int q_tiles, int total, cudaStream_t stream) {
  auto kernel = attention_f8_tile_kernel<HD>;
  constexpr int SMEM_BYTES = Shape<HD>::TILE_BYTES + (int)sizeof(Misc);
  static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "attention_f8_tile: %s", cudaGetErrorString(e));
    configured.done();
  }
  const int sms = tc_host::sm_count();
  return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3((unsigned)(total < sms ? total : sms)), dim3(THREADS), SMEM_BYTES, stream, dim3(1), km, vm, p,
                                             q_tiles, total), "attention_f8_tile");
}

}  // namespace

// Heads of 64 or 128, pages of 16, 32, 64 or 128 keys, up to 128 query heads a group; for requests of more than decode_rows(g) rows (new tokens
// times heads of a group), the others are left.
GB_EXPORT int gb_f8_attention_tile(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale, const void* table,
                                   int table_width, const void* cu_q, const void* kv_lens, void* out, int R, long long pages, int Hq, int Hkv, int hd,
                                   float scale, int window, int page, int max_q_len, void* stream) {
  if (R <= 0 || Hkv <= 0 || Hq % Hkv || (hd != 64 && hd != 128) || page < 16 || page > 128 || (page & (page - 1)) || Hq / Hkv > QROWS ||
      (uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)k_pool % 16 || (uintptr_t)v_pool % 16)
    return gb::fail(GB_BAD_ARGUMENT, "attention_f8_tile: %d requests, heads %d / %d of %d, pages of %d", R, Hq, Hkv, hd, page);
  CUtensorMap km, vm;
  int rc = pool_map(k_pool, page, Hkv, pages, hd, &km);
  if (rc) return rc;
  rc = pool_map(v_pool, page, Hkv, pages, hd, &vm);
  if (rc) return rc;
  const int g = Hq / Hkv, tokens_per_tile = QROWS / g, q_tiles = (max_q_len + tokens_per_tile - 1) / tokens_per_tile;
  const long long total = (long long)q_tiles * Hkv * R;
  if (total > 0x7fffffff) return gb::fail(GB_UNSUPPORTED, "attention_f8_tile: %lld pieces of work", total);
  const Params p{(const __nv_bfloat16*)q, (const float*)k_scale, (const float*)v_scale, (__nv_bfloat16*)out, (const int32_t*)table,
                 (const int32_t*)cu_q, (const int32_t*)kv_lens, table_width, R, Hq, Hkv, g, window, page, scale * 1.4426950408889634f};
  const cudaStream_t st = (cudaStream_t)stream;
  return hd == 64 ? launch<64>(p, km, vm, q_tiles, (int)total, st) : launch<128>(p, km, vm, q_tiles, (int)total, st);
}

GB_EXPORT int gb_f8_attention_tile_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_f8_attention_tile_set_error_sink(void* host_word) { return gb_err::set_sink((int*)host_word); }
