// Matrix product in 8 bits: out[m, n] = sum over blocks b of 128 channels of
//     sa[m, b] * sw[n / 128, b] * sum_{k in b} a8[m, k] w8[n, k],
// codes in E4M3, scales powers of two: one per token and block for the tokens, one per 128 x 128 block for the weights.
//
// The scales are the tensor cores' own: tcgen05.mma of kind mxf8f6f4 multiplies every 32 channels of a row by a power of two that lies in
// tensor memory (a byte, the exponent), so that one accumulator in tensor memory takes all of K. (With scales applied outside, every
// block's 128 x 256 sums have to come back through registers: that form of this kernel took 1.6 us a block and pair of CTAs, five times
// what the products take.) Four products of 32 channels share a block's byte; a 32-bit word holds a row's bytes of four
// blocks, which the instruction chooses from, so scales are brought in once in four blocks.
//
// The weights' rows are the rows of the products (128 a CTA), the tokens their columns, up to 240 a tile: a weight is fetched once for
// all of a tile's tokens, and a step of a few tokens multiplies no padding but to 16.
//
// Tiles are dealt in turn to the workers (a CTA, or a pair of CTAs) while there is a whole round of them, neighbours (the same weights, other
// tokens) at the same time, so that L2 holds what is in use. What is left is dealt in units of (tile, block), an equal stretch
// to every worker: few tokens on a wide weight are bound by how evenly the weights' bytes are shared out, and many tokens leave no ragged
// last round. A tile that falls to several workers is summed by the one that finishes last: each writes its part to scratch memory and
// counts itself; the last adds the parts in the order of the channels, whoever it is, so that results do not depend on the order of arrival.
//
// PAIR: two CTAs of a cluster multiply 256 weight rows by up to 240 tokens (cta_group::2), each fetching half of the tokens' codes.
//   warp 0     TMA: a box of 128 bytes (128 channels) by 128 weight rows and one by the tokens, a ring of stages. Weights are asked for
//              before the wait for the kernel in front, which makes the codes.
//   warp 1     one elected lane: scales into tensor memory, four products a unit
//   warps 2, 3 the scales of four blocks into shared memory: row r's word at 16 (r % 32) + 4 (r / 32) of 512 bytes for 128 rows, as
//              the copy to tensor memory wants it (128 equal words for the weights, whose scale belongs to the block)
//   warps 4-11 at a tile's end: write out, or write the part and perhaps add the parts up; the products go on in the
//              other of two accumulators
// Every wait is bounded.
#include "float8.cuh"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

#include <cmath>

namespace {

using namespace tc;

constexpr int BK = f8::BLOCK;                   // channels per unit: 128 bytes, one swizzled row
constexpr int BM = 128;                         // weight rows per CTA
constexpr int MAX_NT = 240;                     // tokens per tile: two accumulators leave room for the scales
constexpr int THREADS = 128 + 256;
constexpr int MAX_STAGES = 12;
constexpr int SF_STAGES = 4, SF_BYTES = 3 * 512;        // the weights' words, the tokens' (up to 256)
constexpr int SMEM_LIMIT = 232448, STATIC_BYTES = 1024;
// tensor memory: accumulators at columns 0 and 256, scales in the gaps behind them: two sets in turn, so that copying one set does not wait
// for the products that read the other
constexpr uint32_t ACC_STRIDE = 256, SFA_COL = 240, SFB_COL = 244;

struct Args {
  const uint32_t* xs;       // [ceil(blocks / 4)][M]: the tokens' scales, four blocks' exponents a word
  const float* ws;          // [ceil(N / 128)][blocks]: the weights'
  void* out;                // [M, N]
  float* parts;             // scratch: [workers][2][CTAs of a worker][nt][128]
  int* counters;            // [tiles * CTAs of a worker], zero between launches
  int M, N, blocks;
  int nt, tiles_m;          // tokens per tile (a multiple of 16), tiles of tokens
  int stages;               // of one unit, or (STEP) two
  int workers, rounds;      // rounds: whole tiles for every worker
  long long units;          // those of the tiles behind the rounds,
  int share;                // and the workers that share these
  float alpha;
};

// kind mxf8f6f4, both operands E4M3 and K-major, scales UE8M0 (bit 23), one per row and 32 channels; sums in 32 bits. `id`: which byte of
// the scales' words (the same for both operands).
__device__ __forceinline__ uint32_t instr_desc_mxf8(int m, int n, uint32_t id) {
  return (id << 4) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) | (id << 29);
}
template <bool PAIR>
__device__ __forceinline__ void mma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
        : "memory");
}
// 512 bytes of shared memory (32 rows of 16 bytes) to four columns of tensor memory, the 32 rows to the lanes of every warp.
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Rows of 16 bytes one behind the other, eight to a group of 128 bytes, not swizzled.
__device__ __forceinline__ uint64_t smem_desc_rows16(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// The exponent byte of a scale; 255 (not a number) for one that is no positive power of two.
__device__ __forceinline__ uint32_t scale_byte(float s) {
  const uint32_t bits = __float_as_uint(s);
  return (bits & 0x807FFFFFu) == 0 && bits != 0 ? bits >> 23 : 255u;
}

// Where a worker's stretch of units begins.
__host__ __device__ inline long long first_unit(long long units, int workers, int w) { return units * w / workers; }
// The worker whose stretch holds unit u.
__device__ __forceinline__ int worker_of(long long units, int workers, long long u) {
  int w = (int)(u * workers / units);
  while (w + 1 < workers && first_unit(units, workers, w + 1) <= u) ++w;
  while (w > 0 && first_unit(units, workers, w) > u) --w;
  return w;
}

// A worker's walk: tiles worker, worker + workers, ... of the rounds, then its stretch of the rest.
struct Walk {
  int tile, b, i, n;          // where it is; units done, units in all
  int rest_tile, rest_b, tile0, in_rounds, blocks, step;
  __device__ __forceinline__ void start(const Args& p, int worker) {
    blocks = p.blocks, step = p.workers, tile0 = p.rounds * p.workers, in_rounds = p.rounds * p.blocks;
    const long long from = worker < p.share ? first_unit(p.units, p.share, worker) : 0, to = worker < p.share ? first_unit(p.units, p.share, worker + 1) : 0;
    rest_tile = tile0 + (int)(from / blocks), rest_b = (int)(from % blocks);
    i = 0, n = in_rounds + (int)(to - from);
    tile = p.rounds > 0 ? worker : rest_tile, b = p.rounds > 0 ? 0 : rest_b;
  }
  __device__ __forceinline__ bool more() const { return i < n; }
  __device__ __forceinline__ int left() const { return min(blocks - b, n - i); }               // units of it from here on
  __device__ __forceinline__ void advance(int k) {       // by up to left()
    i += k, b += k;
    if (b < blocks) return;
    b = 0;
    if (tile >= tile0) ++tile;
    else if ((tile += step) >= tile0) tile = rest_tile, b = rest_b;
  }
};

template <bool PAIR, int STEP, typename OT, bool ADD>
__global__ void __launch_bounds__(THREADS, 1)
gemm_f8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const Args p) {
  constexpr int CTAS = PAIR ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], sf_full[SF_STAGES], sf_empty[SF_STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s, last_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int worker = blockIdx.x / CTAS;
  const int x_rows = p.nt / CTAS;                                  // rows of the tokens' box
  const uint32_t unit_bytes = (uint32_t)(BM + x_rows) * BK, stage_bytes = unit_bytes * STEP;        // a stage: weights, then tokens
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int stages = p.stages;
  const uint32_t sf_at = ring + stages * stage_bytes;              // behind the ring: the scales on their way
  Walk q;
  q.start(p, worker);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int s = 0; s < SF_STAGES; ++s) {
      mbar_init(smem_u32(&sf_full[s]), CTAS);
      mbar_init(smem_u32(&sf_empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&acc_full[a]), 1);
      mbar_init(smem_u32(&acc_empty[a]), 8 * CTAS);
    }
    abort_s = 0;
    fence_barrier_init();
    fence_proxy_async();
    prefetch_tensormap(&w_map);
    prefetch_tensormap(&x_map);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(&tmem_base_s), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_base_s), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_arrive_wait();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base_s;
  volatile int* aborted = &abort_s;
  gb::pdl_launch_dependents();

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    // What does not change within a tile is worked out once a tile, here and in the issuer: a division a step and a look at the abort flag
    // made a step 650 cycles, whatever its width.
    const bool leader = elect_one();
    bool go = true;
    struct Rows {
      int w, x;              // the first weight row and token of the tile that this CTA fetches
    };
    auto rows_of = [&](const Walk& at) {
      const int n = at.tile / p.tiles_m;
      return Rows{(n * CTAS + (int)rank) * BM, (at.tile - n * p.tiles_m) * p.nt + (int)rank * x_rows};
    };
    auto load_w = [&](int s, int b, int n, int row) {          // n blocks
      const uint32_t full = smem_u32(&full_bar[s]), bar = PAIR ? map_to_rank(full, 0) : full, to = ring + s * stage_bytes;
      if (rank == 0) mbar_arrive_expect_tx(full, n * CTAS * unit_bytes);
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        if (k >= n) break;
        if (PAIR) tma_load_2d_pair(to + k * (BM * BK), &w_map, bar, (b + k) * BK, row);
        else tma_load_2d(to + k * (BM * BK), &w_map, bar, (b + k) * BK, row);
      }
    };
    auto load_x = [&](int s, int b, int n, int row) {
      const uint32_t full = smem_u32(&full_bar[s]), bar = PAIR ? map_to_rank(full, 0) : full, to = ring + s * stage_bytes + STEP * (BM * BK);
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        if (k >= n) break;
        if (PAIR) tma_load_2d_pair(to + k * (x_rows * BK), &x_map, bar, (b + k) * BK, row);
        else tma_load_2d(to + k * (x_rows * BK), &x_map, bar, (b + k) * BK, row);
      }
    };
    // the first stages' weights before the wait for the kernel that makes the codes
    Walk ahead = q;
    for (int i = 0; i < stages && ahead.more(); ++i) {
      const int n = min(STEP - (ahead.b & (STEP - 1)), ahead.left()), row = rows_of(ahead).w;
      if (leader) load_w(i, ahead.b, n, row);
      ahead.advance(n);
    }
    __syncwarp();
    gb::pdl_wait();
    for (int i = 0; i < stages && q.more(); ++i) {
      const int n = min(STEP - (q.b & (STEP - 1)), q.left()), row = rows_of(q).x;
      if (leader) load_x(i, q.b, n, row);
      q.advance(n);
    }
    __syncwarp();
    int s = 0, par = 0;
    while (q.more() && go) {
      const Rows row = rows_of(q);
      const int all = q.left(), b_end = q.b + all;
      for (int b = q.b; b < b_end;) {
        const int n = min(STEP - (b & (STEP - 1)), b_end - b);
        if (!(go = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty_bar[s]), par)))) {
          gb_err::report(ERR_WAIT_EMPTY), *aborted = 1;
          break;
        }
        if (leader) load_w(s, b, n, row.w), load_x(s, b, n, row.x);
        if (++s == stages) s = 0, par ^= 1;
        b += n;
      }
      q.advance(all);
    }
    __syncwarp();
    if (leader && *aborted && q.n > 0) {
      // wind down: the copies in flight need microseconds to land; two milliseconds before the shared memory is given up
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {}
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // -------------------------------------------------------------- the products' issuer
      const uint32_t idesc0 = instr_desc_mxf8(CTAS * BM, p.nt, 0);
      const uint64_t da0 = smem_desc_sw128(ring), db0 = smem_desc_sw128(ring + STEP * (BM * BK)), ds0 = smem_desc_rows16(sf_at);
      const uint32_t stage_step = stage_bytes >> 4, x_step = (uint32_t)(x_rows * BK) >> 4;
      const bool leader = elect_one(), wide = p.nt > 128;
      int s = 0, par = 0, sf = 0, sf_par = 0, failed = 0;
      uint32_t set = ACC_STRIDE, at = 0;          // the set of scales; the stage, in units of the descriptors
      for (int t = 0; q.more() && !failed; ++t) {      // tiles, or parts of them
        const int as = t & 1, n = q.left(), b_end = q.b + n;
        const uint32_t acc = tmem + as * ACC_STRIDE;
        if (!mbar_wait(smem_u32(&acc_empty[as]), ((t >> 1) & 1) ^ 1)) failed = ERR_WAIT_ACCUM;        // both epilogue groups have read it
        for (int b = q.b; b < b_end && !failed;) {
          const int blocks = min(STEP - (b & (STEP - 1)), b_end - b);
          if (b == q.b || (b & 3) == 0) {    // the scales of up to four blocks
            if (!mbar_wait(smem_u32(&sf_full[sf]), sf_par)) failed = ERR_WAIT_FULL;
            tc_fence_after_sync();
            set ^= ACC_STRIDE;
            if (leader && !failed) {
              const uint64_t ds = ds0 + (uint64_t)(sf * (SF_BYTES >> 4));
              copy_scales<PAIR>(tmem + set + SFA_COL, ds);
              copy_scales<PAIR>(tmem + set + SFB_COL, ds + (512 >> 4));
              if (wide) copy_scales<PAIR>(tmem + set + SFB_COL + 4, ds + (1024 >> 4));
              if (PAIR) mma_commit_pair(smem_u32(&sf_empty[sf]), 3);
              else mma_commit(smem_u32(&sf_empty[sf]));
            }
            if (++sf == SF_STAGES) sf = 0, sf_par ^= 1;
          }
          if (!mbar_wait(smem_u32(&full_bar[s]), par)) failed = ERR_WAIT_FULL;
          tc_fence_after_sync();
          if (leader && !failed) {
            uint64_t da = da0 + at, db = db0 + at;
#pragma unroll
            for (int i = 0; i < STEP; ++i, da += (BM * BK) >> 4, db += x_step) {
              if (i >= blocks) break;
              const uint32_t id = (uint32_t)((b + i) & 3), idesc = idesc0 | (id << 4) | (id << 29);
#pragma unroll
              for (int k = 0; k < BK / 32; ++k)
                mma_mxf8<PAIR>(acc, da + 2 * k, db + 2 * k, idesc, tmem + set + SFA_COL, tmem + set + SFB_COL, b + i > q.b || k > 0);
            }
            if (PAIR) mma_commit_pair(smem_u32(&empty_bar[s]), 3);
            else mma_commit(smem_u32(&empty_bar[s]));
          }
          at += stage_step;
          if (++s == stages) s = 0, par ^= 1, at = 0;
          b += blocks;
        }
        if (leader && !failed) {
          if (PAIR) mma_commit_pair(smem_u32(&acc_full[as]), 3);
          else mma_commit(smem_u32(&acc_full[as]));
        }
        __syncwarp();
        q.advance(n);
      }
      if (failed) {
        gb_err::report(failed);
        *aborted = 1;
      }
    }
  } else if (warp == 2 || warp == 3) {
    // ---------------------------------------------------------------- scales
    // Two warps, every second four blocks each. The next ones are asked for once the current ones have been handed over: the fence in front of
    // that waits for loads under way. (One warp that asked for them before took 2,200 cycles for four blocks, more than their products.)
    bool ran_out;
    gb::pdl_wait();          // the tokens' scales
    uint32_t x[8];           // this lane's tokens lane, 32 + lane, ...
    float w = 0.f;           // lanes 0 to 3: the weights' blocks
    bool there = false;
    auto ask = [&](const Walk& at) {
      const int n = at.tile / p.tiles_m, m0 = (at.tile - n * p.tiles_m) * p.nt, nb = n * CTAS + (int)rank, g = at.b >> 2, wb = 4 * g + lane;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = j * 32 + lane;
        x[j] = c < p.nt && m0 + c < p.M ? p.xs[(size_t)g * p.M + m0 + c] : 0u;
      }
      there = lane < 4 && wb < p.blocks && nb * BM < p.N;
      w = there ? p.ws[(size_t)nb * p.blocks + wb] : 0.f;
    };
    auto next = [&]() { q.advance(min(4 - (q.b & 3), q.left())); };
    int turn = 0;            // fours so far
    if (warp == 3 && q.more()) next(), ++turn;
    if (q.more()) ask(q);
    while (q.more()) {
      const int sf = turn % SF_STAGES;
      uint32_t put_w = there ? scale_byte(w) << (8 * lane) : 0u;
      put_w |= __shfl_xor_sync(0xffffffffu, put_w, 1);
      put_w |= __shfl_xor_sync(0xffffffffu, put_w, 2);
      put_w = __shfl_sync(0xffffffffu, put_w, 0);
      if (!mbar_wait_warp(smem_u32(&sf_empty[sf]), (turn / SF_STAGES & 1) ^ 1, aborted, ran_out)) {
        if (ran_out) gb_err::report(ERR_WAIT_EMPTY), *aborted = 1;
        break;
      }
      uint4* to = reinterpret_cast<uint4*>(smem_raw + (sf_at - smem_u32(smem_raw)) + sf * SF_BYTES) + lane;
      to[0] = make_uint4(put_w, put_w, put_w, put_w);
      to[32] = make_uint4(x[0], x[1], x[2], x[3]);
      to[64] = make_uint4(x[4], x[5], x[6], x[7]);
      fence_proxy_async();            // the tensor core reads them through the async proxy
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) mbar_arrive(smem_u32(&sf_full[sf]));
        else mbar_arrive_cluster(map_to_rank(smem_u32(&sf_full[sf]), 0));
      }
      next();
      if (q.more()) next();
      turn += 2;
      if (q.more()) ask(q);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- results
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    // this group's columns of a tile: half of them, in whole sixteens
    const int half = (p.nt / 16 + 1) / 2 * 16, col0 = group * half, cols = group ? p.nt - half : half;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16) + col0;
    gb::pdl_wait();          // for ADD the output; and the scratch that the launch in front may still read
    bool ok = true;
#pragma unroll 1
    for (int t = 0; q.more(); ++t) {
      const int as = t & 1;
      const int n = q.left();          // units of this part
      const bool whole = n == p.blocks;
      const int row = (q.tile / p.tiles_m * CTAS + (int)rank) * BM + quarter * 32 + lane;
      const int m0 = q.tile % p.tiles_m * p.nt + col0;
      const int have = min(cols, p.M - m0);
      OT* out = reinterpret_cast<OT*>(p.out) + (size_t)m0 * p.N + row;
      // what is added to, sixteen columns ahead of its turn (read where it is needed, a column's latency stood behind every other's: an added
      // product of 2,048 x 2,048 x 2,048 took 70 us, a plain one 19)
      float old[16], ahead[16];
      auto ask = [&](int c0, float (&x)[16]) {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = ADD && row < p.N && c0 + e < have ? gb::to_float(out[(size_t)(c0 + e) * p.N]) : 0.f;
      };
      auto keep = [&] {
#pragma unroll
        for (int e = 0; e < 16; ++e) old[e] = ahead[e];
      };
      if (whole) ask(0, ahead);
      if (ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[as]), (t >> 1) & 1) && !*aborted);
        if (!ok) {                // from here on this warp only keeps the others company at the barriers
          if (lane == 0 && !*aborted) gb_err::report(ERR_WAIT_ACCUM);
          *aborted = 1;
        }
      }
      tc_fence_after_sync();
      auto put = [&](int c, float x, float before) { out[(size_t)c * p.N] = gb::from_float<OT>(ADD ? fmaf(p.alpha, x, before) : x); };
      const size_t part_floats = (size_t)p.nt * BM;
      auto part_of = [&](int w, int which) {
        return p.parts + ((size_t)(w * 2 + which) * CTAS + rank) * part_floats + (size_t)col0 * BM + quarter * 32 + lane;
      };
      float* my = part_of(worker, q.i == q.in_rounds ? 0 : 1);
      if (ok) {
#pragma unroll 1
        for (int c0 = 0; c0 < cols; c0 += 16) {
          uint32_t v[16];
          tmem_ld_16(lane_addr + as * ACC_STRIDE + c0, v);
          if (ADD && whole) {
            keep();
            ask(c0 + 16, ahead);
          }
          tmem_ld_wait();
          if (whole) {
            if (row < p.N) {
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (c0 + e < have) put(c0 + e, __uint_as_float(v[e]), old[e]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c0 + e < have) my[(size_t)(c0 + e) * BM] = __uint_as_float(v[e]);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) mbar_arrive(smem_u32(&acc_empty[as]));
          else mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[as]), 0));
        }
      }
      if (!whole) {
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int rest = q.tile - q.tile0;
        const long long t0 = (long long)rest * p.blocks;
        const int first = worker_of(p.units, p.share, t0), last = worker_of(p.units, p.share, t0 + p.blocks - 1);
        if (threadIdx.x == 128) {
          int* counter = p.counters + (size_t)rest * CTAS + rank;
          const int before = atomicAdd(counter, 1);
          last_s = before == last - first;
          if (last_s) *counter = 0;          // as the next launch expects it
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (last_s && ok && row < p.N) {
          __threadfence();
          // of the workers that share the tile only the first may have begun in front of it. Sixteen columns at a time, all of a
          // part's loads under way at once.
          const int which = (int)(first_unit(p.units, p.share, first) / p.blocks) == rest ? 0 : 1;
#pragma unroll 1
          for (int c0 = 0; c0 < have; c0 += 16) {
            float sum[16];
            ask(c0, old);
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[e] = c0 + e < have ? __ldcg(part_of(first, which) + (size_t)(c0 + e) * BM) : 0.f;
#pragma unroll 2
            for (int w = first + 1; w <= last; ++w) {
              const float* part = part_of(w, 0) + (size_t)c0 * BM;
#pragma unroll
              for (int e = 0; e < 16; ++e) sum[e] += c0 + e < have ? __ldcg(part + (size_t)e * BM) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c0 + e < have) put(c0 + e, sum[e], old[e]);
          }
        }
        // (the flag is read before a next part's first barrier, and written behind it)
      }
      q.advance(n);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_arrive_wait();       // neither CTA leaves while the other's products or copies may touch it
  if (warp == 1) {
    if (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ host side
struct MapKey {
  const void* ptr;
  long long rows, cols, pitch;
  int box;
  bool operator==(const MapKey& o) const {
    return ptr == o.ptr && rows == o.rows && cols == o.cols && pitch == o.pitch && box == o.box;
  }
};
struct MapKeyHash {
  size_t operator()(const MapKey& k) const {
    return std::hash<const void*>()(k.ptr) ^ (std::hash<long long>()(k.rows) * 31) ^ (std::hash<long long>()(k.cols) * 131) ^
           (std::hash<long long>()(k.pitch) * 521) ^ (size_t)k.box * 7919;
  }
};

// [rows, cols] bytes, rows `pitch` apart, through boxes of `box` rows x 128 bytes with the 128-byte swizzle; outside it
// is zeros. (A map says where a matrix lies and how long it is, not what it holds.)
int tensor_map(const void* ptr, long long rows, long long cols, long long pitch, int box_rows, CUtensorMap* out) {
  static std::mutex mu;
  static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
  const MapKey key{ptr, rows, cols, pitch, box_rows};
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(key);
  if (it != cache.end()) {
    *out = it->second;
    return GB_OK;
  }
  tc_host::EncodeTiledFn fn = tc_host::encode_fn();
  if (!fn) return gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUtensorMap m;
  const CUresult r = fn(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
                        estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled failed with code %d for a %lld x %lld matrix of codes", (int)r, rows, cols);
  if (cache.size() > 4096) cache.clear();
  cache.emplace(key, m);
  *out = m;
  return GB_OK;
}

struct Plan {
  bool pair;
  int nt, stages, step, workers, rounds, share;
  int tiles_m, tiles_n;
  long long units;          // of the tiles behind the rounds
};

// Shared memory for the stages. Three of two units fit for every pair of CTAs, whose units hold half of the tokens: pairs come with two
// units to a stage only.
constexpr int ROOM_BYTES = SMEM_LIMIT - 1024 - STATIC_BYTES - SF_STAGES * SF_BYTES;
static_assert(3 * 2 * (BM + MAX_NT / 2) * BK <= ROOM_BYTES, "a pair's stages");

// What a product of this shape would take, in microseconds, with `tiles` tiles of tokens, in pairs or not: the plan and its time, from what
// was measured here. An SM takes in 115 KB a microsecond from L2, all together 11 MB, and 6.4 MB from memory; a step of a unit takes the issuing warp
// 0.26 us (two units to a stage: 0.15 each), products of 256 tokens 0.27; a part of a tile costs its bytes once out and once in, and
// 1.2 us each way; a pair of CTAs starts and ends 1.5 us later. The results of a tile's end overlap the next tile's products.
Plan plan_of(int M, int N, int K, int tiles, bool pair, double* us_out) {
  Plan q;
  q.pair = pair;
  q.nt = ((M + tiles - 1) / tiles + 15) / 16 * 16;
  q.tiles_m = (M + q.nt - 1) / q.nt;
  const int ctas = pair ? 2 : 1, blocks = (K + BK - 1) / BK;
  q.tiles_n = (N + BM * ctas - 1) / (BM * ctas);
  const long long tiles_all = (long long)q.tiles_m * q.tiles_n, units = tiles_all * blocks;
  const int unit = (BM + q.nt / ctas) * BK;
  q.step = ROOM_BYTES / (2 * unit) >= 3 ? 2 : 1;           // two units to a stage where three such stages fit (4096 x 28672 x 4096: 354 us against 386)
  q.stages = ROOM_BYTES / (q.step * unit) < MAX_STAGES ? ROOM_BYTES / (q.step * unit) : MAX_STAGES;
  const int room = tc_host::sm_count() / ctas;
  q.workers = (int)(units < room ? units : room);
  q.rounds = (int)(tiles_all / q.workers);
  const auto unit_us = [&](double active) {
    const double fetch = fmax(unit / 115e3, active * ctas * unit / 11e6), memory = active * ctas * BM * BK / 6.4e6 / q.tiles_m;
    return fmax(fmax(fetch, memory), fmax(q.step == 2 ? 0.15 : 0.26, 0.27 * q.nt / 256));
  };
  const double rounds_us = (double)q.rounds * blocks * unit_us(q.workers) + (pair ? 1.5 : 0.0);
  // the tiles that are left, each among c workers
  const long long rest = tiles_all - (long long)q.rounds * q.workers;
  q.units = rest * blocks;
  q.share = 0;
  double best = rest > 0 ? 1e30 : 0;
  for (int c = 1; rest > 0 && c <= 16; ++c) {
    const long long all = rest * c < q.workers ? rest * c : q.workers, share = all < q.units ? all : q.units;
    const double units_each = (double)((q.units + share - 1) / share);
    const double parts = share > rest ? (rest * c <= q.workers ? c : (double)share / rest + 1) + 1 : 0;
    const double us = units_each * unit_us((double)share) + parts * (1.2 + (double)(M < q.nt ? M : q.nt) * BM * 4 / 67e3);
    if (us < best) best = us, q.share = (int)share;
    if (all == q.workers) break;
  }
  *us_out = rounds_us + best;
  return q;
}

Plan make_plan(int M, int N, int K) {
  const int least = (M + MAX_NT - 1) / MAX_NT;
  double us, best = 1e30;
  Plan plan{};
  for (int pair = 0; pair < 2; ++pair)
    for (int tiles = least; tiles <= least + 3 && tiles <= (M + 15) / 16; ++tiles) {
      const Plan q = plan_of(M, N, K, tiles, pair != 0, &us);
      if (us < best) best = us, plan = q;
    }
  return plan;
}

long long code_bytes(int M, int K) { return ((long long)M * ((K + 15) / 16 * 16) + 255) / 256 * 256; }
long long scale_bytes(int M, int K) { return ((long long)(K + 4 * BK - 1) / (4 * BK) * M * 4 + 255) / 256 * 256; }
long long part_bytes(const Plan& q) { return (long long)(q.share > 0 ? q.share : 1) * 2 * (q.pair ? 2 : 1) * q.nt * BM * 4; }
long long counter_bytes(const Plan& q) { return ((long long)q.tiles_m * q.tiles_n * (q.pair ? 2 : 1) * 4 + 255) / 256 * 256; }

template <bool PAIR, int STEP, typename OT, bool ADD>
int launch(const Plan& q, const CUtensorMap& wm, const CUtensorMap& xm, const Args& a, cudaStream_t stream) {
  auto kernel = gemm_f8_kernel<PAIR, STEP, OT, ADD>;
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - STATIC_BYTES);
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "gemm_f8: %s", cudaGetErrorString(e));
    configured.done();
  }
  const int ctas = PAIR ? 2 : 1;
  const size_t smem = (size_t)q.stages * STEP * (BM + q.nt / ctas) * BK + SF_STAGES * SF_BYTES + 1024;
  return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3((unsigned)(q.workers * ctas)), dim3(THREADS), smem, stream, dim3(ctas), wm, xm, a),
                              "gemm_f8");
}

template <bool PAIR, int STEP>
int launch_out(const Plan& q, const CUtensorMap& wm, const CUtensorMap& xm, const Args& a, int out_tag, bool add, cudaStream_t stream) {
  if (add) return launch<PAIR, STEP, float, true>(q, wm, xm, a, stream);
  if (out_tag == GB_F32) return launch<PAIR, STEP, float, false>(q, wm, xm, a, stream);
  return launch<PAIR, STEP, __nv_bfloat16, false>(q, wm, xm, a, stream);
}

}  // namespace

int gb_f8_quantize_rows(const void* a, int tag, long long lda, int gated, int M, int K, void* codes, int pitch, void* scales, cudaStream_t stream);

// Bytes of scratch that a product of this shape wants (codes, scales and parts; no need to clear them), and of counters (zero before the
// first launch; every launch leaves them zero).
GB_EXPORT long long gb_f8_linear_scratch_bytes(int M, int N, int K, long long* counters) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan q = make_plan(M, N, K);
  *counters = counter_bytes(q);
  return code_bytes(M, K) + scale_bytes(M, K) + part_bytes(q);
}

// How a product of this shape is cut: CTAs of a worker, units of a stage, tokens of a tile, tiles, workers, rounds of whole tiles, and of the tiles
// behind these the workers that share them.
GB_EXPORT int gb_f8_linear_plan(int M, int N, int K, int* out) {
  if (M <= 0 || N <= 0 || K <= 0) return gb::fail(GB_BAD_ARGUMENT, "linear_float8_plan: %d x %d x %d", M, N, K);
  const Plan q = make_plan(M, N, K);
  const int values[7] = {q.pair ? 2 : 1, q.step, q.nt, q.tiles_m * q.tiles_n, q.workers, q.rounds, q.share};
  for (int i = 0; i < 7; ++i) out[i] = values[i];
  return GB_OK;
}

// out [M, N] (+)= q(a) w^T: a [M, K] with rows lda apart (gated: [M, 2 K], rows [gate | up], multiplied as silu(gate) * up), w [N, K] codes
// with rows w_pitch apart, ws its scales.
GB_EXPORT int gb_f8_linear(const void* a, int a_tag, long long lda, const void* w, long long w_pitch, const void* ws, void* out, int out_tag, int M,
                           int N, int K, int accumulate, float alpha, int gated, void* counters, void* scratch, void* stream) {
  if (M < 0 || N < 0 || K <= 0) return gb::fail(GB_BAD_ARGUMENT, "linear_float8: %d x %d x %d", M, N, K);
  if (M == 0 || N == 0) return GB_OK;
  if (w_pitch % 16 || w_pitch < K || (uintptr_t)w % 16 || (uintptr_t)scratch % 256)
    return gb::fail(GB_BAD_ARGUMENT, "linear_float8: rows of codes start on 16 bytes (pitch %lld)", w_pitch);
  if (accumulate && out_tag != GB_F32) return gb::fail(GB_BAD_ARGUMENT, "linear_float8: accumulates into 32 bits only");
  const cudaStream_t st = (cudaStream_t)stream;
  const int pitch = (K + 15) / 16 * 16;
  uint8_t* codes = (uint8_t*)scratch;
  uint8_t* xs = codes + code_bytes(M, K);
  int rc = gb_f8_quantize_rows(a, a_tag, lda, gated, M, K, codes, pitch, xs, st);
  if (rc) return rc;
  const Plan q = make_plan(M, N, K);
  const int ctas = q.pair ? 2 : 1;
  CUtensorMap wm, xm;
  rc = tensor_map(w, N, K, w_pitch, BM, &wm);
  if (rc) return rc;
  rc = tensor_map(codes, M, pitch, pitch, q.nt / ctas, &xm);
  if (rc) return rc;
  const Args args{(const uint32_t*)xs, (const float*)ws, out, (float*)(xs + scale_bytes(M, K)), (int*)counters, M, N, (K + BK - 1) / BK, q.nt,
                  q.tiles_m, q.stages, q.workers, q.rounds, q.units, q.share, accumulate ? alpha : 1.0f};
  const bool add = accumulate != 0;
  if (q.pair) return launch_out<true, 2>(q, wm, xm, args, out_tag, add, st);
  return q.step == 2 ? launch_out<false, 2>(q, wm, xm, args, out_tag, add, st) : launch_out<false, 1>(q, wm, xm, args, out_tag, add, st);
}

GB_EXPORT int gb_f8_gemm_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_f8_gemm_set_error_sink(void* host_word) { return gb_err::set_sink((int*)host_word); }
