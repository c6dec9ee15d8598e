// Matrix product in 8 bits: out[m, n] = sum over blocks b of 128 channels of
//     sa[m, b] * sw[n / 128, b] * sum_{k in b} a8[m, k] w8[n, k],
// codes in E4M3, scales in 32 bits: one per token and block for the tokens, one per 128 x 128 block for the weights.
//
// The weights' rows are the rows of the products (128 a CTA), the tokens their columns: up to 256, so that a weight is fetched once for
// up to 256 tokens, and a step of a few tokens multiplies no padding but to 16. tcgen05.mma (kind::f8f6f4, 32 channels each, sums in 32
// bits) leaves a block's sums in tensor memory; as every block has scales of its own, sums of several blocks cannot stay there:
// eight warps read a block's 128 x tokens sums back and add them, scaled, to accumulators in registers, while the tensor cores
// fill the other of two buffers. A lane holds a weight row, so the scales of a step are the same for all lanes: they are
// multiplied (token's by weight's), put into shared memory by the warp that uses them, and read four at a time.
//
// Work is dealt in units of (tile, block), tile by tile, an equal stretch to every CTA (or pair of CTAs): few tokens on a wide
// weight are bound by how evenly the weights' bytes are shared out, and many tokens leave no ragged last round. A tile that falls to
// several CTAs is summed by the one that finishes last: each writes its part to scratch memory and counts itself; the last adds the
// parts in the order of the channels, whoever it is, so that results do not depend on the order of arrival.
//
// PAIR: two CTAs of a cluster multiply 256 weight rows by up to 256 tokens (cta_group::2), each fetching half of the tokens' codes.
//   warp 0     TMA: a box of 128 bytes (128 channels) by 128 weight rows and one by the tokens, a ring of stages. Weights are asked for
//              before the wait for the kernel in front, which makes the codes.
//   warp 1     one elected lane: four products a unit, one commit (the stage's "empty" barrier is passed on by the epilogue: a commit
//              costs the issuing lane as much as two products)
//   warps 2-9  scale and add; at a tile's end write out, or write the part and perhaps add the parts up
// Every wait is bounded.
#include "float8.cuh"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace {

using namespace tc;

constexpr int BK = f8::BLOCK;                   // channels per unit: 128 bytes, one swizzled row
constexpr int BM = 128;                         // weight rows per CTA
constexpr int THREADS = 64 + 256;
constexpr int MAX_STAGES = 12;
constexpr int SMEM_LIMIT = 232448;

struct Args {
  const float* xs;          // [blocks][M]: the tokens' scales
  const float* ws;          // [ceil(N / 128)][blocks]: the weights'
  void* out;                // [M, N]
  float* parts;             // scratch: [workers][2][CTAs of a worker][nt][128]
  int* counters;            // [tiles * CTAs of a worker], zero between launches
  int M, N, blocks;
  int nt, tiles_m;          // tokens per tile (a multiple of 16; PAIR: of 32), tiles of tokens
  int stages, workers;
  long long units;
  float alpha;
};

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Sums in 32 bits, both operands E4M3 and K-major.
__device__ __forceinline__ uint32_t instr_desc_e4m3(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[N]);
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t addr, uint32_t (&r)[32]) { tmem_ld_32(addr, r); }
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t addr, uint32_t (&r)[16]) { tmem_ld_16(addr, r); }
template <>
__device__ __forceinline__ void tmem_load<8>(uint32_t addr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr)
               : "memory");
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

// CH: tokens per epilogue thread (each of the two groups of four warps takes CH of the tile's columns, the second what is left)
template <bool PAIR, int CH, typename OT, bool ADD>
__global__ void __launch_bounds__(THREADS, 1)
gemm_f8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const Args p) {
  constexpr int CTAS = PAIR ? 2 : 1;
  constexpr int CHUNK = CH % 32 == 0 ? 32 : CH % 16 == 0 ? 16 : 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s, last_s;
  __shared__ __align__(16) float scale_s[8][2][CH];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int worker = blockIdx.x / CTAS;
  const int x_rows = p.nt / CTAS;                                  // rows of the tokens' box
  const uint32_t stage_bytes = (uint32_t)(BM + x_rows) * BK;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const long long u_begin = first_unit(p.units, p.workers, worker), u_end = first_unit(p.units, p.workers, worker + 1);
  const int n_units = (int)(u_end - u_begin);
  const int stages = p.stages;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
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
    const bool leader = elect_one();
    bool go = true, ran_out;
    struct Place { int tile, b; } at = {(int)(u_begin / p.blocks), (int)(u_begin % p.blocks)};
    auto next = [&](Place& q) {
      if (++q.b == p.blocks) q.b = 0, ++q.tile;
    };
    auto load_w = [&](int s, const Place& q) {
      const uint32_t full = smem_u32(&full_bar[s]), bar = PAIR ? map_to_rank(full, 0) : full;
      const int row = (q.tile / p.tiles_m * CTAS + (int)rank) * BM;
      if (rank == 0) mbar_arrive_expect_tx(full, CTAS * stage_bytes);
      if (PAIR) tma_load_2d_pair(ring + s * stage_bytes, &w_map, bar, q.b * BK, row);
      else tma_load_2d(ring + s * stage_bytes, &w_map, bar, q.b * BK, row);
    };
    auto load_x = [&](int s, const Place& q) {
      const uint32_t full = smem_u32(&full_bar[s]), bar = PAIR ? map_to_rank(full, 0) : full;
      const int row = q.tile % p.tiles_m * p.nt + (int)rank * x_rows;
      if (PAIR) tma_load_2d_pair(ring + s * stage_bytes + BM * BK, &x_map, bar, q.b * BK, row);
      else tma_load_2d(ring + s * stage_bytes + BM * BK, &x_map, bar, q.b * BK, row);
    };
    // the first stages' weights before the wait for the kernel that makes the codes
    const int early = min(stages, n_units);
    Place q = at;
    for (int i = 0; i < early; ++i, next(q))
      if (leader) load_w(i, q);
    __syncwarp();
    gb::pdl_wait();
    q = at;
    for (int i = 0; i < early; ++i, next(q))
      if (leader) load_x(i, q);
    __syncwarp();
    int s = 0, par = 0;
    for (int i = early; i < n_units && go; ++i, next(q)) {
      if (!(go = mbar_wait_warp(smem_u32(&empty_bar[s]), par, aborted, ran_out))) {
        if (ran_out) gb_err::report(ERR_WAIT_EMPTY), *aborted = 1;
        break;
      }
      if (leader) load_w(s, q), load_x(s, q);
      __syncwarp();
      if (++s == stages) s = 0, par ^= 1;
    }
    if (leader && *aborted && n_units > 0) {
      // wind down: the copies in flight need microseconds to land; two milliseconds before the shared memory is given up
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {}
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // -------------------------------------------------------------- the products' issuer
      const uint32_t idesc = instr_desc_e4m3(CTAS * BM, p.nt);
      const uint64_t da0 = smem_desc_sw128(ring), db0 = smem_desc_sw128(ring + BM * BK);
      const bool leader = elect_one();
      bool go = true, ran_out;
      int s = 0, par = 0;
      for (int i = 0; i < n_units && go; ++i) {
        const int as = i & 1;
        if (!(go = mbar_wait_warp(smem_u32(&acc_empty[as]), ((i >> 1) & 1) ^ 1, aborted, ran_out))) {
          if (ran_out) gb_err::report(ERR_WAIT_ACCUM), *aborted = 1;
          break;
        }
        if (!(go = mbar_wait_warp(smem_u32(&full_bar[s]), par, aborted, ran_out))) {
          if (ran_out) gb_err::report(ERR_WAIT_FULL), *aborted = 1;
          break;
        }
        tc_fence_after_sync();
        const uint64_t da = da0 + (uint64_t)(s * (stage_bytes >> 4)), db = db0 + (uint64_t)(s * (stage_bytes >> 4));
        if (leader) {
#pragma unroll
          for (int k = 0; k < BK / 32; ++k) {
            if (PAIR) mma_f8_pair(tmem + as * 256, da + 2 * k, db + 2 * k, idesc, k > 0);
            else mma_f8(tmem + as * 256, da + 2 * k, db + 2 * k, idesc, k > 0);
          }
          if (PAIR) mma_commit_pair(smem_u32(&acc_full[as]), 3);
          else mma_commit(smem_u32(&acc_full[as]));
        }
        __syncwarp();
        if (++s == stages) s = 0, par ^= 1;
      }
    }
  } else {
    // ---------------------------------------------------------------- scale, add, write
    const int ew = warp - 2, quarter = warp & 3, group = ew >> 2;
    const int col0 = group * CH, cols = max(0, min(CH, p.nt - col0));        // this group's columns of the tile
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16) + col0;
    const bool passes_on = threadIdx.x == 64;
    float acc[CH];
    gb::pdl_wait();          // the scales and, for ADD, the output
    int tile = (int)(u_begin / p.blocks), b = (int)(u_begin % p.blocks), from = b;
    int i = 0, s = 0;
    // the scales of a unit: this lane's tokens' and the weight block's
    constexpr int PER = (CH + 31) / 32;
    float mine[PER];
    auto fetch = [&](int t, int blk) {
      const int m0 = t % p.tiles_m * p.nt + col0, nb = t / p.tiles_m * CTAS + (int)rank;
      const float w = (nb * BM < p.N) ? p.ws[(size_t)nb * p.blocks + blk] : 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int c = j * 32 + lane;
        mine[j] = (c < cols && m0 + c < p.M) ? p.xs[(size_t)blk * p.M + m0 + c] * w : 0.f;
      }
    };
    if (n_units > 0) fetch(tile, b);
    bool ok = true;
    for (; i < n_units; ++i) {
      const int as = i & 1;
      if (b == from) {
#pragma unroll
        for (int c = 0; c < CH; ++c) acc[c] = 0.f;
      }
      float* sc = scale_s[ew][as];
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (j * 32 + lane < CH) sc[j * 32 + lane] = mine[j];
      __syncwarp();
      const bool tile_ends = b + 1 == p.blocks;
      if (i + 1 < n_units) fetch(tile_ends ? tile + 1 : tile, tile_ends ? 0 : b + 1);
      if (ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[as]), (i >> 1) & 1) && !*aborted);
        if (!ok) {                // from here on this warp only keeps the others company at the barriers
          if (lane == 0 && !*aborted) gb_err::report(ERR_WAIT_ACCUM);
          *aborted = 1;
        }
      }
      tc_fence_after_sync();
      if (passes_on && ok) mbar_arrive(smem_u32(&empty_bar[s]));       // the products have read the stage
      if (++s == stages) s = 0;
#pragma unroll
      for (int c0 = 0; c0 < CH; c0 += CHUNK) {
        if (c0 >= cols || !ok) break;
        uint32_t v[CHUNK];
        tmem_load<CHUNK>(lane_addr + as * 256 + c0, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < CHUNK; e += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sc + c0 + e);
          acc[c0 + e] = fmaf(__uint_as_float(v[e]), f.x, acc[c0 + e]);
          acc[c0 + e + 1] = fmaf(__uint_as_float(v[e + 1]), f.y, acc[c0 + e + 1]);
          acc[c0 + e + 2] = fmaf(__uint_as_float(v[e + 2]), f.z, acc[c0 + e + 2]);
          acc[c0 + e + 3] = fmaf(__uint_as_float(v[e + 3]), f.w, acc[c0 + e + 3]);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0 && ok) {
        if (rank == 0) mbar_arrive(smem_u32(&acc_empty[as]));
        else mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[as]), 0));
      }
      if (tile_ends || i + 1 == n_units) {
        // ---- the end of a tile, or of this worker's part of it
        const int row = (tile / p.tiles_m * CTAS + (int)rank) * BM + quarter * 32 + lane;
        const int m0 = tile % p.tiles_m * p.nt + col0;
        const int have = min(cols, p.M - m0);
        const bool whole = tile_ends && from == 0;
        bool write = whole;
        if (!whole) {
          const size_t part_floats = (size_t)p.nt * BM;
          auto part_of = [&](int w, int which) {
            return p.parts + ((size_t)(w * 2 + which) * CTAS + rank) * part_floats + (size_t)col0 * BM + quarter * 32 + lane;
          };
          const long long t0 = (long long)tile * p.blocks;
          float* my = part_of(worker, tile == (int)(u_begin / p.blocks) ? 0 : 1);
#pragma unroll
          for (int c = 0; c < CH; ++c)
            if (c < have) my[(size_t)c * BM] = acc[c];
          __threadfence();
          asm volatile("bar.sync 1, 256;" ::: "memory");
          const int first = worker_of(p.units, p.workers, t0), last = worker_of(p.units, p.workers, t0 + p.blocks - 1);
          if (threadIdx.x == 64) {
            int* counter = p.counters + (size_t)tile * CTAS + rank;
            const int before = atomicAdd(counter, 1);
            last_s = before == last - first;
            if (last_s) *counter = 0;          // as the next launch expects it
          }
          asm volatile("bar.sync 1, 256;" ::: "memory");
          write = last_s != 0;
          if (write) {
            __threadfence();
#pragma unroll
            for (int c = 0; c < CH; ++c) acc[c] = 0.f;
            for (int w = first; w <= last; ++w) {
              const float* part = part_of(w, (int)(first_unit(p.units, p.workers, w) / p.blocks) == tile ? 0 : 1);
#pragma unroll
              for (int c = 0; c < CH; ++c)
                if (c < have) acc[c] += __ldcg(part + (size_t)c * BM);
            }
          }
        }
        if (write && ok && row < p.N) {
          OT* out = reinterpret_cast<OT*>(p.out) + (size_t)m0 * p.N + row;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            if (c < have) {
              OT* to = out + (size_t)c * p.N;
              if (ADD) *to = gb::from_float<OT>(fmaf(p.alpha, acc[c], gb::to_float(*to)));
              else *to = gb::from_float<OT>(acc[c]);
            }
          }
        }
        from = 0;
      }
      if (tile_ends) b = 0, ++tile;
      else ++b;
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
  int box_rows;
  bool operator==(const MapKey& o) const {
    return ptr == o.ptr && rows == o.rows && cols == o.cols && pitch == o.pitch && box_rows == o.box_rows;
  }
};
struct MapKeyHash {
  size_t operator()(const MapKey& k) const {
    return std::hash<const void*>()(k.ptr) ^ (std::hash<long long>()(k.rows) * 31) ^ (std::hash<long long>()(k.cols) * 131) ^
           (std::hash<long long>()(k.pitch) * 521) ^ (size_t)k.box_rows * 7919;
  }
};

// [rows, cols] bytes, rows `pitch` apart, through boxes of box_rows x 128 bytes with the 128-byte swizzle; outside it is zeros. (A map
// says where a matrix lies and how long it is, not what it holds.)
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
  const CUresult r = fn(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return gb::fail(GB_CUDA_ERROR, "cuTensorMapEncodeTiled failed with code %d for a %lld x %lld matrix of codes", (int)r, rows, cols);
  if (cache.size() > 4096) cache.clear();
  cache.emplace(key, m);
  *out = m;
  return GB_OK;
}

struct Plan {
  bool pair;
  int nt, ch, stages, workers;
  int tiles_m, tiles_n;
  long long units;
};

Plan make_plan(int M, int N, int K) {
  Plan q;
  q.pair = M > 512;
  const int tiles = (M + 255) / 256, step = q.pair ? 32 : 16;
  q.nt = ((M + tiles - 1) / tiles + step - 1) / step * step;
  q.tiles_m = (M + q.nt - 1) / q.nt;
  const int ctas = q.pair ? 2 : 1, blocks = (K + BK - 1) / BK;
  q.tiles_n = (N + BM * ctas - 1) / (BM * ctas);
  q.units = (long long)q.tiles_m * q.tiles_n * blocks;
  const int half = (q.nt + 1) / 2;
  q.ch = half <= 8 ? 8 : half <= 16 ? 16 : half <= 32 ? 32 : half <= 64 ? 64 : half <= 96 ? 96 : 128;
  const int stage = (BM + q.nt / ctas) * BK;
  const int most = (SMEM_LIMIT - 1024 - 2048 - 8 * 2 * q.ch * 4) / stage;
  q.stages = most < MAX_STAGES ? most : MAX_STAGES;
  const int room = tc_host::sm_count() / ctas;
  q.workers = (int)(q.units < room ? q.units : room);
  return q;
}

long long part_bytes(const Plan& q) { return (long long)q.workers * 2 * (q.pair ? 2 : 1) * q.nt * BM * 4; }
long long counter_bytes(const Plan& q) { return ((long long)q.tiles_m * q.tiles_n * (q.pair ? 2 : 1) * 4 + 255) / 256 * 256; }

template <bool PAIR, int CH, typename OT, bool ADD>
int launch(const Plan& q, const CUtensorMap& wm, const CUtensorMap& xm, const Args& a, cudaStream_t stream) {
  auto kernel = gemm_f8_kernel<PAIR, CH, OT, ADD>;
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - 2048 - 8 * 2 * CH * 4);
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "gemm_f8: %s", cudaGetErrorString(e));
    configured.done();
  }
  const int ctas = PAIR ? 2 : 1;
  const size_t smem = (size_t)q.stages * (BM + q.nt / ctas) * BK + 1024;
  return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3((unsigned)(q.workers * ctas)), dim3(THREADS), smem, stream, dim3(ctas), wm, xm, a),
                              "gemm_f8");
}

template <bool PAIR, int CH>
int launch_out(const Plan& q, const CUtensorMap& wm, const CUtensorMap& xm, const Args& a, int out_tag, bool add, cudaStream_t stream) {
  if (add) return launch<PAIR, CH, float, true>(q, wm, xm, a, stream);
  if (out_tag == GB_F32) return launch<PAIR, CH, float, false>(q, wm, xm, a, stream);
  return launch<PAIR, CH, __nv_bfloat16, false>(q, wm, xm, a, stream);
}

}  // namespace

// Bytes of scratch a product of this shape wants: counters (zero before the first launch; every launch leaves them zero) and parts.
GB_EXPORT long long gb_f8_gemm_scratch_bytes(int M, int N, int K, long long* counters) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan q = make_plan(M, N, K);
  *counters = counter_bytes(q);
  return part_bytes(q);
}

GB_EXPORT int gb_f8_gemm(const void* codes, int pitch, const void* xs, const void* w, long long w_pitch, const void* ws, void* out, int out_tag,
                         int M, int N, int K, int accumulate, float alpha, void* counters, void* parts, void* stream) {
  if (M < 0 || N < 0 || K <= 0) return gb::fail(GB_BAD_ARGUMENT, "gemm_f8: %d x %d x %d", M, N, K);
  if (M == 0 || N == 0) return GB_OK;
  if (w_pitch % 16 || w_pitch < K || (uintptr_t)w % 16 || (uintptr_t)codes % 16 || pitch % 16 || pitch < K)
    return gb::fail(GB_BAD_ARGUMENT, "gemm_f8: rows of codes start on 16 bytes (pitches %d and %lld)", pitch, w_pitch);
  if (accumulate && out_tag != GB_F32) return gb::fail(GB_BAD_ARGUMENT, "gemm_f8: accumulates into 32 bits only");
  const Plan q = make_plan(M, N, K);
  const int ctas = q.pair ? 2 : 1;
  CUtensorMap wm, xm;
  int rc = tensor_map(w, N, K, w_pitch, BM, &wm);
  if (rc) return rc;
  rc = tensor_map(codes, M, pitch, pitch, q.nt / ctas, &xm);
  if (rc) return rc;
  Args a{(const float*)xs, (const float*)ws, out, (float*)parts, (int*)counters, M, N, (K + BK - 1) / BK, q.nt, q.tiles_m, q.stages,
         q.workers, q.units, accumulate ? alpha : 1.0f};
  const cudaStream_t st = (cudaStream_t)stream;
  const bool add = accumulate != 0;
  if (q.pair) return launch_out<true, 128>(q, wm, xm, a, out_tag, add, st);
  switch (q.ch) {
    case 8: return launch_out<false, 8>(q, wm, xm, a, out_tag, add, st);
    case 16: return launch_out<false, 16>(q, wm, xm, a, out_tag, add, st);
    case 32: return launch_out<false, 32>(q, wm, xm, a, out_tag, add, st);
    case 64: return launch_out<false, 64>(q, wm, xm, a, out_tag, add, st);
    case 96: return launch_out<false, 96>(q, wm, xm, a, out_tag, add, st);
    default: return launch_out<false, 128>(q, wm, xm, a, out_tag, add, st);
  }
}

GB_EXPORT int gb_f8_gemm_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_f8_gemm_set_error_sink(void* host_word) { return gb_err::set_sink((int*)host_word); }
