// Attention of prompt portions over pages of E4M3 codes with a scale per page and head, on the fifth-generation tensor cores.
//
//   s_j = (q . k8_j) * ks(page of j) * scale over keys [start, pos];  out = sum_j softmax(s)_j vs(page of j) v8_j
// (garuda/src/llama/mod.rs:793-818; the window garuda/src/cache/mod.rs:333-338; query head h reads key/value head h / g).
//
// A piece of work is 256 query rows, (token, head-of-group) pairs of one kv head of one request, in two halves of 128; its keys are walked in
// tiles of 128. The kernel is persistent: one CTA per SM takes pieces until none are left (rounds of gridDim.x pieces, walked forth and
// back so that long and short ones mix). Per half: S = Q K^T into tensor memory, a softmax in registers (a thread has a row and all 128 keys
// of the tile), P back over S, O += P V; while one half's softmax runs, the tensor cores work for the other. Products run in the order of
// their issue, so a half's next S, which overwrites P, is issued right behind the P V that reads it, and the end of an S product says that
// the P V in front has ended too: the accumulator may be rescaled without another wait.
// (The bfloat16 kernel's arrangement, 128 rows whose tiles two groups share and S two tiles ahead, took 70 us for 2,048 tokens of 32 heads of 128
// and 105 us for two portions of 509 over a window of 4,096; this one takes 55 and 79, that kernel itself 59 and 92.) A tile takes 4,000
// clocks: a half's softmax is 2,200 of them, 1,500 for the exponentials (1,024 at their pipe's rate), and 1,900 pass from its weights to
// its next scores (1,024 of products at the tensor cores' rate): the halves' chains, not a unit, set the pace. Two threads a row, sixteen
// softmax warps, took 61 and 96; 32 scores at a time in a loop 63 and 94; a quarter of the exponentials as polynomials 63 and 85.
//   * S is a product of codes as they lie (tcgen05.mma kind f8f6f4): a query row, scaled by a power of two to a largest of at most 448, is the
//     sum of two E4M3 rows (a bfloat16's eight bits are four and four: exact down to 2^-9 of the row's largest; what is below that
//     loses bits, and is gone below 2^-17: both products add to the same sums, so the second row cannot have a finer unit), so
//     S = Qhi K^T + Qlo K^T at twice the rate of bfloat16: the same time, half of the keys' bytes.
//   * Values become halves (exactly: every E4M3 number is one) in shared memory, a conversion for two of them, by four warps of
//     their own, for 256 rows' worth of products. (Splitting P into codes instead would cost the softmax warps two instructions a score.)
//   * A page's ks goes into the factor of the exponent's multiply-add, its vs (as a power of two) into the constant; the denominator takes it
//     out again per sixteen keys. P in halves: eleven bits, down to 2^-30 of what a row refers to, its own largest weight times vs: a
//     page that a row may not read, or whose keys have no weight, takes no bits from the others however large its values are.
//   * The references follow the running maxima only when one has been outgrown by 2^8 for some row of a warp.
//   warp 0      TMA: keys and values, a box a page, into rings of their own; looks up pages and scales four tiles at a time, two steps ahead
//   warp 1      one elected lane issues the products
//   warps 4-11  softmax, four warps a half; their half's queries of the next piece as codes; results
//   warps 12-15 the values of the next tile as halves (rows that no query reads as zeros)
// Registers are shared out by need (setmaxnreg; with 184 for the softmax some went to memory, and it took 60 us). Every wait is bounded.
#include "attention_float8.cuh"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace {

using namespace tc;
using namespace attn8;

constexpr int QROWS = 256;          // query rows per CTA
constexpr int HALF = 128;           // of a half
constexpr int KT = 128;             // keys per tile
constexpr int BLOCK_BYTES = 128 * 128;              // 128 values' rows of one block of 64 channels in halves
constexpr int TMEM_COLS = 512;
constexpr int O_COL0 = 2 * KT;                      // behind the halves' S
constexpr int THREADS = 512;
constexpr float RESCALE_ABOVE = 8.f;                // in powers of two
constexpr float UP = 6.f;                           // probabilities are multiplied by 2^6: halves go to 65,504, and down to 2^-30 of the reference
constexpr int SLOTS = 16;                            // tiles' scales in flight
// registers a thread of the warpgroups: copies and products, softmax (two), conversions; 128 a thread at launch
constexpr int REGS_ISSUE = 56, REGS_SOFTMAX = 200, REGS_CONVERT = 56;
static_assert(REGS_ISSUE + 2 * REGS_SOFTMAX + REGS_CONVERT <= 4 * 128, "no more registers than at launch");

template <int HD>
struct Shape {
  static constexpr int BLOCKS = HD / 64;                              // blocks of 64 channels of values in halves
  static constexpr int Q_BYTES = 2 * QROWS * HD, CODE_BYTES = KT * HD, H_BYTES = BLOCKS * BLOCK_BYTES;
  static constexpr int K_STAGES = HD == 64 ? 4 : 3, V_STAGES = HD == 64 ? 4 : 2, H_STAGES = HD == 64 ? 3 : 2;
  static constexpr int K_AT = Q_BYTES, V_AT = K_AT + K_STAGES * CODE_BYTES, H_AT = V_AT + V_STAGES * CODE_BYTES;
  static constexpr int TILE_BYTES = H_AT + H_STAGES * H_BYTES;
  static_assert(O_COL0 + 2 * HD <= TMEM_COLS, "tensor memory layout");
  static_assert(K_STAGES + 5 <= SLOTS, "a tile's scales outlive its keys");
};

// Barriers and the like, behind the tiles in dynamic shared memory.
struct Misc {
  uint64_t q_full[2], k_full[6], k_empty[6], v_full[4], v_empty[4], h_full[3], h_empty[3];
  uint64_t s_ready[2], p_ready[2][2], o_ready[2], o_free[2];
  uint32_t tmem_base;
  int abort;
  float2 scales[SLOTS][8];              // a tile's ks of each sixteen keys (negative: no page there) and log2 of vs
  float factor[QROWS];                  // per query row: 2^e * scale * log2(e)
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// Two at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// One piece of work: 256 query rows of one request and kv head.
struct Item {
  bool valid;
  int kvh, q_begin, tok0, nrows, pos0, lo, hi, tile_begin, n_tiles;
  const int32_t* table;
  // tiles of a half: the first rows of a piece see fewer keys than the last
  __device__ __forceinline__ int tiles_of(int half, int g) const {
    const int rows = min(HALF, nrows - half * HALF);
    if (rows <= 0) return 0;
    return max(1, (pos0 + (half * HALF + rows - 1) / g) / KT + 1 - tile_begin);
  }
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
  const int kv_len = p.kv_lens[r];
  const int ntok = min(tokens_per_tile, q_len - w.tok0);
  w.nrows = ntok * p.g;
  w.pos0 = kv_len - q_len + w.tok0;                                 // position of the tile's first token
  w.lo = p.window > 0 ? max(0, w.pos0 + 1 - p.window) : 0;          // first key any row reads
  w.hi = w.pos0 + ntok - 1;                                         // last key any row reads
  w.tile_begin = w.lo / KT;
  w.valid = q_len * p.g > decode_rows(p.g) && w.tok0 < q_len && w.hi >= w.lo;      // else a decode request, or past its end
  w.n_tiles = w.valid ? w.hi / KT + 1 - w.tile_begin : 0;
  w.table = p.block_table + (size_t)r * p.table_width;
  return w;
}

// The k-th item of this CTA: rounds of gridDim.x items, walked forth and back in turn, so that the
// CTA that got the longest item of one round gets the shortest of the next.
__device__ __forceinline__ int cta_item(int k) {
  const int g = (int)gridDim.x, b = (int)blockIdx.x;
  return k * g + ((k & 1) ? g - 1 - b : b);
}

// Walks this CTA's items.
struct Cursor {
  int item, total, step, q_tiles, round;
  int it;          // valid items before this one
  int j;           // tile within the item (for who walks tiles)
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
// halves' tiles, and everything it executes delays the tensor cores. Its lanes decode 32 items at
// a time, one each; the walk then only shuffles the counts out.
struct CountWalk {
  int base;        // this CTA's items before the batch
  int my_n[2];     // tiles of the halves of this lane's item of the batch (0: none, or not a valid item)
  int lane_i;      // the next item's lane
  int n[2];
  __device__ __forceinline__ void load(const Params& p, int q_tiles, int total) {
    const int k = base + (int)(threadIdx.x & 31);
    const long long item = (long long)k * gridDim.x < total ? cta_item(k) : total;
    my_n[0] = my_n[1] = 0;
    if (item < total) {
      const Item w = decode_item(p, q_tiles, (int)item);
      if (w.valid) my_n[0] = w.tiles_of(0, p.g), my_n[1] = w.tiles_of(1, p.g);
    }
  }
  __device__ __forceinline__ void start(const Params& p, int q_tiles, int total) {
    base = 0, lane_i = 0;
    load(p, q_tiles, total);
  }
  // The next item's counts; false: there is none.
  __device__ __forceinline__ bool next(const Params& p, int q_tiles, int total) {
    for (;;) {
      const unsigned have = lane_i < 32 ? __ballot_sync(0xffffffffu, my_n[0] > 0) & (0xffffffffu << lane_i) : 0u;
      if (have != 0) {
        const int l = __ffs(have) - 1;
        n[0] = __shfl_sync(0xffffffffu, my_n[0], l), n[1] = __shfl_sync(0xffffffffu, my_n[1], l);
        lane_i = l + 1;
        return true;
      }
      base += 32, lane_i = 0;
      if ((long long)base * gridDim.x >= total) return false;
      load(p, q_tiles, total);
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
  const uint32_t q_s = smem_u32(smem_raw);                         // the rows' codes, then what they leave
  const uint32_t k_s = q_s + S::K_AT, v_s = q_s + S::V_AT, h_s = q_s + S::H_AT;
  if ((q_s & 1023u) != 0) {                                        // the swizzle needs it; never seen
    if (threadIdx.x == 0) gb_err::report(ERR_WAIT_DRAIN);
    return;
  }

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&mc.q_full[b]), 128);
      mbar_init(smem_u32(&mc.s_ready[b]), 2);       // the product's end; the issuing thread, who has seen the keys' scales arrive
      mbar_init(smem_u32(&mc.p_ready[b][0]), 128);
      mbar_init(smem_u32(&mc.p_ready[b][1]), 128);
      mbar_init(smem_u32(&mc.o_ready[b]), 1);
      mbar_init(smem_u32(&mc.o_free[b]), 128);
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
  // Queries, scales and this step's keys and values come from the kernel in front (pdl_wait below); the batch's lengths and block tables were
  // there before the step's first kernel.
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
      gb::pdl_wait();
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
          if (mine) mc.scales[gt % SLOTS][sub] = make_float2(now.ks, fmaxf(log2f(now.vs), -100.f));
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
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = instr_desc(HALF, KT), idesc_o = instr_desc(HALF, HD) | INSTR_B_MN_MAJOR;
      const uint64_t dq0 = smem_desc_rows<HD>(q_s), dk0 = smem_desc_rows<HD>(k_s), dv0 = smem_desc_sw128_mn(h_s, BLOCKS > 1 ? BLOCK_BYTES : 16);
      bool ok = true;
      int ks = 0, kpar = 0, hs = 0, hpar = 0;       // stages (and phases) of the keys and values in use
      int sp[2] = {0, 0}, used[2] = {0, 0};                  // phases of p_ready, items so far, a half each
      auto wait = [&](uint64_t& bar, int par, int code) {
        if (!ok) return;
        const bool came = mbar_wait(smem_u32(&bar), par);
        if (!came) gb_err::report(code);
        ok = __all_sync(0xffffffffu, came);
      };
      CountWalk w;
      w.start(p, q_tiles, total_items);
      while (ok && w.next(p, q_tiles, total_items)) {
        const int n0 = w.n[0], n1 = w.n[1], n = max(n0, n1);
        auto issue_s = [&](int h, int j) {       // S = (Qhi + Qlo) K^T of tile j
          const bool first = h == 0, last = h == 1 || j >= n1;       // of the halves that read these keys
          if (first || j >= n0) wait(mc.k_full[ks], kpar, ERR_WAIT_FULL);
          tc_fence_after_sync();
          if (leader && ok) {
            const uint64_t dq = dq0 + (uint64_t)(h * HALF * HD >> 4), dk = dk0 + (uint64_t)(ks * (S::CODE_BYTES >> 4));
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int k = 0; k < HD / 32; ++k)
                mma_f8(tmem_base + h * KT, dq + (uint64_t)(part * (QROWS * HD >> 4) + 2 * k), dk + 2 * k, idesc_s, part > 0 || k > 0);
            mbar_arrive(smem_u32(&mc.s_ready[h]));
            mma_commit(smem_u32(&mc.s_ready[h]));
            if (last) mma_commit(smem_u32(&mc.k_empty[ks]));
          }
          __syncwarp();
          if (last && ++ks == K_STAGES) ks = 0, kpar ^= 1;
        };
        wait(mc.q_full[0], used[0] & 1, ERR_WAIT_FULL);
        issue_s(0, 0);
        if (n1 > 0) {
          wait(mc.q_full[1], used[1] & 1, ERR_WAIT_FULL);
          issue_s(1, 0);
        }
        for (int j = 0; j < n && ok; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int mine = h == 0 ? n0 : n1;
            if (j >= mine) continue;
            const bool last = h == 1 || j >= n1;                     // of the halves that read these values
            if (j == 0 && used[h] > 0) wait(mc.o_free[h], (used[h] - 1) & 1, ERR_WAIT_ACCUM);        // the item in front has been written out
            if (j == 0) ++used[h];
            if (h == 0 || j >= n0) wait(mc.h_full[hs], hpar, ERR_WAIT_FULL);
            const uint64_t dv = dv0 + (uint64_t)(hs * (S::H_BYTES >> 4));
#pragma unroll
            for (int k = 0; k < KT / 64; ++k) {              // 64 keys' weights at a time, while the softmax is at the next
              wait(mc.p_ready[h][k], sp[h], ERR_WAIT_ACCUM);
              tc_fence_after_sync();
              if (leader && ok)
                mma_bf16_ts<4>(tmem_base + O_COL0 + h * HD, tmem_base + h * KT + k * 32, dv + (uint64_t)(k * (64 * 128 >> 4)), idesc_o,
                               16 * 128 >> 4, j > 0 || k > 0);
              __syncwarp();
            }
            sp[h] ^= 1;
            if (leader && ok) {
              if (last) mma_commit(smem_u32(&mc.h_empty[hs]));
              if (j == mine - 1) mma_commit(smem_u32(&mc.o_ready[h]));
            }
            __syncwarp();
            if (last && ++hs == H_STAGES) hs = 0, hpar ^= 1;
            if (j + 1 < mine) issue_s(h, j + 1);
          }
        }
      }
      if (!ok) *abort_s = 1;
    }
  } else if (warp >= 12) {
    // -------------------------------------------------------------------- conversions
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONVERT));
    const int x = threadIdx.x - 384;             // a key
    bool ok = true;
    int gt = 0, vs = 0, vpar = 0, hs = 0, hpar = 1;
    Cursor c;
    for (c.start(p, q_tiles, total_items); !c.done && ok; c.next_item(p)) {
      const Item& w = c.w;
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
        const uint32_t keep = readable ? 0xffffffffu : 0u;
#pragma unroll 2
        for (int i = 0; i < HD / 16; ++i) {          // sixteen channels: two chunks of halves
          const uint4 code = *reinterpret_cast<const uint4*>(from + swizzled<HD>(x, i));
          const uint32_t u[4] = {code.x & keep, code.y & keep, code.z & keep, code.w & keep};
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
      }
    }
  } else {
    // -------------------------------------------------------------------- softmax warps
    // Warps 4-7 have the first half's rows, 8-11 the second's: a thread a row.
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int half = (warp - 4) >> 2;
    const int quarter = warp & 3;                        // the TMEM lanes this warp may read
    const int row = half * HALF + quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + half * KT, o_addr = lane_addr + O_COL0 + half * HD;
    bool ok = true;
    int gt = 0, sph = 0, oph = 0;          // tiles so far (all items' and both halves'), phases of s_ready and o_ready
    bool ran_out = false;
    // The queries of an item as codes: this warp's 32 rows, eight channels a lane. (Nobody reads the old ones any more: the product of the
    // half's last tile has been waited for.)
    auto put_queries = [&](const Cursor& at) {
      const Item& w = at.w;
      if (at.done || w.nrows <= half * HALF) return;
      constexpr int LANES = HD / 8, ROWS = 32 / LANES, BATCH = 8;          // lanes of a row, rows of a load
      const int sub = lane % LANES, row0 = half * HALF + quarter * 32 + lane / LANES;
      const int own_row = (w.q_begin + w.tok0 + row / p.g) * p.Hq + w.kvh * p.g + row % p.g;          // of `q`
#pragma unroll 1
      for (int i0 = 0; i0 < 32 / ROWS; i0 += BATCH) {
        uint4 raw[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int from = __shfl_sync(0xffffffffu, own_row, (i0 + i) * ROWS + lane / LANES);
          raw[i] = row0 + (i0 + i) * ROWS < w.nrows ? *reinterpret_cast<const uint4*>(p.q + (size_t)from * HD + sub * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int qr = row0 + (i0 + i) * ROWS;
          const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          uint32_t hi[2], lo[2];
          const float unit = split_query<LANES>(u, 1.f, hi, lo);
          uint8_t* to = smem_raw + swizzled<HD>(qr, sub >> 1) + (sub & 1) * 8;
          *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(to + QROWS * HD) = make_uint2(lo[0], lo[1]);
          if (sub == 0) mc.factor[qr] = unit * p.scale_log2;
        }
      }
      fence_proxy_async();              // the tensor core reads them through the async proxy
      mbar_arrive(smem_u32(&mc.q_full[half]));
      __syncwarp();
    };
    Cursor next;                           // the item after the current one
    next.start(p, q_tiles, total_items);
    gb::pdl_wait();
    Item w{};                              // the current one
    int n = 0;                             // its tiles of this half
    // the references, in powers of two: of scores (the denominator's unit), of weights times vs (the accumulators')
    float m = -INFINITY, c = -INFINITY, l = 0.f;
    while (ok) {
      put_queries(next);
      // ---- write the current one out
      if (n > 0) {
        if (!(ok = mbar_wait_warp(smem_u32(&mc.o_ready[half]), oph, abort_s, ran_out))) break;
        oph ^= 1;
        tc_fence_after_sync();
        const float inv = l > 0.f ? exp2_fast(c - m - UP) / l : l == l ? 0.f : l;        // (a score that is no number stays one)
        __nv_bfloat16* dst = p.out + ((size_t)(w.q_begin + w.tok0 + row / p.g) * p.Hq + w.kvh * p.g + row % p.g) * HD;
#pragma unroll 2
        for (int h = 0; h < HD / 16; ++h) {
          uint32_t v[16];
          tmem_ld_16(o_addr + h * 16, v);
          tmem_ld_wait();
          float t[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) t[e] = __uint_as_float(v[e]) * inv;
          if (row < w.nrows) {
            uint4 w0, w1;
            w0.x = pack_bf16(t[0], t[1]), w0.y = pack_bf16(t[2], t[3]), w0.z = pack_bf16(t[4], t[5]), w0.w = pack_bf16(t[6], t[7]);
            w1.x = pack_bf16(t[8], t[9]), w1.y = pack_bf16(t[10], t[11]), w1.z = pack_bf16(t[12], t[13]), w1.w = pack_bf16(t[14], t[15]);
            *reinterpret_cast<uint4*>(dst + h * 16) = w0;
            *reinterpret_cast<uint4*>(dst + h * 16 + 8) = w1;
          }
        }
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&mc.o_free[half]));
      }
      if (next.done) break;
      w = next.w, n = w.tiles_of(half, p.g);
      next.next_item(p);
      m = c = -INFINITY, l = 0.f;
      const int row_pos = row < w.nrows ? w.pos0 + row / p.g : -1;       // no key is valid for a padding row
      const int row_start = (row < w.nrows && p.window > 0) ? max(0, row_pos + 1 - p.window) : 0;
      // what all rows of this half read: up to the first row's position, from the last row's window on
      const int half_lo = w.pos0 + half * HALF / p.g, half_hi = w.pos0 + (min(w.nrows, half * HALF + HALF) - 1) / p.g;
      float factor = 0.f;
      for (int j = 0; j < w.n_tiles; ++j, ++gt) {
        if (j >= n) continue;            // keys that only the other half reads
        if (!(ok = mbar_wait_warp(smem_u32(&mc.s_ready[half]), sph, abort_s, ran_out))) break;
        sph ^= 1;
        tc_fence_after_sync();
        if (j == 0) factor = mc.factor[row];
        uint32_t sv[KT / 32][32];
#pragma unroll
        for (int h = 0; h < KT / 32; ++h) tmem_ld_32(s_addr + h * 32, sv[h]);
        float f[8], ev[8];            // of each sixteen keys: the scores' factor, log2 of vs
        bool pages = true;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const float2 two = mc.scales[gt % SLOTS][b];
          f[b] = two.x * factor, ev[b] = two.y;
          pages = pages && two.x >= 0.f;
        }
        tmem_ld_wait();
        auto sc = [&](int ch) -> float& { return reinterpret_cast<float&>(sv[ch >> 5][ch & 31]); };
        const int key0 = (w.tile_begin + j) * KT;
        // the keys need no mask if they lie wholly before the first row's position and inside the last row's window
        const bool full = pages && key0 + KT - 1 <= half_lo && (p.window <= 0 || key0 >= half_hi + 1 - p.window);
        if (!full) {
#pragma unroll
          for (int h = 0; h < KT / 32; ++h) {          // 32 keys: an interval of bits, less the pages that are not there
            const int first = max(row_start - key0 - 32 * h, 0), end = min(row_pos + 1 - key0 - 32 * h, 32);
            uint32_t bits = end > first ? (0xffffffffu >> (32 - end)) & (0xffffffffu << first) : 0u;
            if (f[2 * h] < 0.f) bits &= 0xffff0000u;
            if (f[2 * h + 1] < 0.f) bits &= 0x0000ffffu;
#pragma unroll
            for (int ch = 0; ch < 32; ++ch)
              if (!(bits >> ch & 1)) sv[h][ch] = 0xff800000u;          // -inf
          }
          // (a factor must not turn a masked score's sign)
#pragma unroll
          for (int b = 0; b < 8; ++b) f[b] = fmaxf(f[b], 0x1p-126f);
        }
        // the maximum of each sixteen keys' raw products, times their factor, and with vs
        float m_new = m, c_new = c;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          float mx = max3(sc(16 * b), sc(16 * b + 1), sc(16 * b + 2));
#pragma unroll
          for (int ch = 3; ch < 15; ch += 2) mx = max3(mx, sc(16 * b + ch), sc(16 * b + ch + 1));
          mx = fmaxf(mx, sc(16 * b + 15));
          m_new = fmaxf(m_new, mx * f[b]), c_new = fmaxf(c_new, fmaf(mx, f[b], ev[b]));
        }
        // The references move only if some row of the warp has outgrown one by more than 2^8; then the warp rescales what it has
        // accumulated (the loads and stores of tensor memory are the whole warp's). A row that has seen no valid key yet has
        // nothing to rescale.
        const bool grown = m != -INFINITY && fmaxf(m_new - m, c_new - c) > RESCALE_ABOVE;
        if (j > 0 && __any_sync(0xffffffffu, grown)) {
          const float own = m == -INFINITY ? 1.f : exp2_fast(m - m_new), corr = m == -INFINITY ? 1.f : exp2_fast(c - c_new);
#pragma unroll 1
          for (int h = 0; h < HD / 16; ++h) {
            uint32_t v[16];
            tmem_ld_16(o_addr + h * 16, v);
            tmem_ld_wait();
#pragma unroll
            for (int ch = 0; ch < 16; ++ch) v[ch] = __float_as_uint(__uint_as_float(v[ch]) * corr);
            tmem_st_16(o_addr + h * 16, v);
          }
          l *= own;
          m = m_new, c = c_new;
        } else if (m == -INFINITY) {
          m = m_new, c = c_new;
        }
        const float neg_m = m == -INFINITY ? 0.f : -m, vref = m == -INFINITY ? 0.f : c - m;       // nothing valid yet: avoid inf - inf
        // (A page's vs counts as 2^-100 of vref at least, which is nothing, so that its keys have numbers for the denominator. Where nothing is
        // read the probabilities are zeros.)
#pragma unroll
        for (int h = 0; h < KT / 32; ++h) {                  // 32 keys: 16 columns of P, over scores that have been read
          uint32_t pk[16];
#pragma unroll
          for (int b = 2 * h; b < 2 * h + 2; ++b) {
            const float up = UP + fmaxf(ev[b] - vref, -100.f), off = neg_m + up;
            const float2 f2 = make_float2(f[b], f[b]), off2 = make_float2(off, off);
            float2 ls = make_float2(0.f, 0.f);
#pragma unroll
            for (int ch = 16 * b; ch < 16 * b + 16; ch += 2) {
              float2 y = fma2(make_float2(sc(ch), sc(ch + 1)), f2, off2);
              y.x = exp2_fast(y.x), y.y = exp2_fast(y.y);                     // exp2(-inf) = 0 for masked keys
              ls = add2(ls, y);
              pk[(ch >> 1) - 16 * h] = pack_f16(y.x, y.y);
            }
            l = fmaf(ls.x + ls.y, exp2_fast(-up), l);          // without vs
          }
          tmem_st_16(s_addr + h * 16, pk);
          if (h == 1) {
            tmem_st_wait();
            tc_fence_before_sync();       // this thread's accesses to tensor memory are over
            mbar_arrive(smem_u32(&mc.p_ready[half][0]));
          }
        }
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&mc.p_ready[half][1]));
      }
    }
    if (!ok) {
      if (ran_out) gb_err::report(ERR_WAIT_ACCUM);
      *abort_s = 1;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// ------------------------------------------------------------------ host side
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
  if (R <= 0 || Hkv <= 0 || Hq % Hkv || (hd != 64 && hd != 128) || page < 16 || page > 128 || (page & (page - 1)) || Hq / Hkv > HALF ||
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
