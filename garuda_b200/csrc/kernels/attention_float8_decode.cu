// Attention of single tokens (few query rows a request) over pages of E4M3 codes with a scale per page and head.
//
//   s_j = (q . k8_j) * ks(page of j) * scale over keys [start, pos];  out = sum_j softmax(s)_j vs(page of j) v8_j
// (garuda/src/llama/mod.rs:793-818; the window garuda/src/cache/mod.rs:333-338; query head h reads key/value head h / g).
//
// Bound by the stream of codes, 2 * HD bytes a key and head: so the codes go from shared memory into the matrix instructions as
// they are (mma.sync m16n8k32 on E4M3; 1.4 of them a nanosecond and SM here, a tile of 32 keys takes 32), and what has more than four
// bits is split instead: a query row, bfloat16 scaled by a power of two to a largest of at most 448, is the sum of two E4M3 rows
// exactly (eight bits of mantissa are four and four; what is 2^-11 of the row's largest and below loses bits that the sum does not
// see), and a weight exp(s - m) * 256 is a code and 1/32 of another, to 2^-9 of itself down to 2^-16 of the largest weight. The two
// parts are rows i and i + 8 of one product, which has 16 rows anyway. Sums, maxima and denominators are 32-bit.
//
// Scales cost nothing per key: a page's ks goes into the factor that the exponent's multiply-add has anyway, its vs (a power of two)
// into the constant of the same; the denominator takes it out again per sixteen keys. The accumulators hold sums in units of the
// largest vs so far.
//
// Work: the tiles (32 keys) of all requests and heads in a row, an equal stretch to every CTA, so that requests of unequal length do
// not wait for the longest. Within a CTA a stretch's tiles go to the warps in turn; every warp has a ring of stages of its own that
// TMA fills (a box per page, swizzled as ldmatrix undoes it), asked for as soon as a stage is free, across the borders of requests.
// At a request's end the warps' sums are merged in shared memory; a request that falls to several CTAs is merged by the one that
// finishes last, in their order, from scratch memory: results do not depend on who that is.
//
// The keys' order within a tile is free (sums run over it), and is chosen so that the scores lie in the lanes where the second product
// wants its weights: slot s of sixteen holds key T(s) = s ^ ((s & 8) >> 2), which also keeps ldmatrix's eight rows on distinct
// banks for keys and for values.
#include "attention_float8.cuh"
#include "error_word.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace {

using namespace tc;
using attn8::Params;

constexpr int TK = 32;                  // keys per tile
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int MAX_ROWS = 16;
constexpr unsigned long long DRAIN_LIMIT_NS = 20000000ull;

template <int HD, int MT>
struct Shape {
  static constexpr int ROWS = 8 * MT;
  static constexpr int OPERAND = TK * HD, STAGE = 2 * OPERAND;          // bytes: keys, values
  static constexpr int DEPTH = 24 * 1024 / STAGE;                       // stages of a warp's ring: 3 or 6
  static constexpr int RING = WARPS * DEPTH * STAGE;                    // 96 KB: two CTAs an SM
  static constexpr int RS = HD + 2;                                     // a row's sums, maximum, denominator: a part in scratch memory
  static constexpr int CW = 64 / MT, PASSES = HD / CW;                  // channels that the warps merge at a time
  static constexpr int MERGE = WARPS * ROWS * CW * 4;                   // 8 KB
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Two 16 x 16 blocks of bytes, transposed: lane l gives row l (of 32); r[0], r[1] hold rows 4 (l % 4) + 0..3 of columns l / 4 and
// 8 + l / 4 of the first block, r[2], r[3] the same of the second.
__device__ __forceinline__ void ldmatrix_trans_bytes(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Byte offset of 16-byte chunk `c` of row `row` in a tile as TMA swizzled it (rows of 128 bytes, or of 64).
template <int HD>
__device__ __forceinline__ uint32_t swizzled(int row, int c) {
  return HD == 128 ? (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}
__device__ __forceinline__ int key_of_slot(int s) { return s ^ ((s & 8) >> 2); }          // within a tile: bit 4 stays

// Two weights (times 256) as a code and 32 times what it leaves, as a code: hi, lo.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  uint16_t h;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(b), "f"(a));
  const uint32_t back = f8::decode2_f16(h);
  uint32_t both, left;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(both) : "f"(b), "f"(a));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(left) : "r"(both), "r"(back));
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(left) : "r"(left), "r"(0x50005000u));          // 32
  uint16_t l;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(l) : "r"(left));
  hi = h, lo = l;
}

// MT: products of eight query rows each (1, or 2 for groups of more than eight heads)
template <int HD, int MT>
__global__ void __launch_bounds__(THREADS, 2)
attention_f8_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Params p,
                           const int box_rows, const int min_tiles, float* __restrict__ partials, int* __restrict__ counters) {
  using S = Shape<HD, MT>;
  constexpr int RS = S::RS, ROWS = S::ROWS, CW = S::CW;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[WARPS * S::DEPTH];
  __shared__ __align__(16) float4 scale_s[WARPS * S::DEPTH];           // a stage's ks of its sixteens (negative: no page), and log2 vs
  __shared__ float2 ml_s[WARPS][ROWS];         // the warps' maxima and denominators
  __shared__ int abort_s, last_s, scan_s[WARPS], total_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  float* red = reinterpret_cast<float*>(ring + S::RING);               // [warps][rows][CW]
  int* cum = reinterpret_cast<int*>(ring + S::RING + S::MERGE);        // [R + 1]: tiles of a head of the requests in front

  if (threadIdx.x == 0) {
    for (int s = 0; s < WARPS * S::DEPTH; ++s) mbar_init(smem_u32(&full_bar[s]), 1);
    abort_s = 0;
    total_s = 0;
    fence_barrier_init();
    fence_proxy_async();
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  __syncthreads();
  gb::pdl_launch_dependents();

  // ---- every request's tiles (the batch's lengths are there before the step's first kernel)
  auto span = [&](int r, int& lo, int& hi, int& pos0, int& nrows) {          // first and last key that any row reads
    const int q_len = p.cu_q[r + 1] - p.cu_q[r], kv_len = p.kv_lens[r];
    nrows = q_len * p.g;
    pos0 = kv_len - q_len;
    lo = p.window > 0 ? max(0, pos0 + 1 - p.window) : 0;
    hi = kv_len - 1;
  };
  for (int r0 = 0; r0 < p.R; r0 += THREADS) {
    const int r = r0 + threadIdx.x;
    int lo, hi, pos0, nrows, n = 0;
    if (r < p.R) {
      span(r, lo, hi, pos0, nrows);
      if (nrows > 0 && nrows <= p.decode_rows && hi >= lo) n = hi / TK - lo / TK + 1;
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan_s[warp] = inc;
    __syncthreads();
    int before = total_s;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
      if (w < warp) before += scan_s[w];
    if (r < p.R) cum[r] = before + inc - n;
    __syncthreads();
    if (threadIdx.x == THREADS - 1) total_s = before + inc;
    __syncthreads();
  }
  if (threadIdx.x == 0) cum[p.R] = total_s;
  __syncthreads();
  const long long tiles = (long long)total_s * p.Hkv;
  // as many CTAs as leave each min_tiles, and no more than share a request's head usefully
  const int workers = (int)max(1ll, min((long long)gridDim.x, tiles / min_tiles));
  const int cta = blockIdx.x;
  if (cta >= workers || tiles == 0) {
    gb::pdl_wait();        // the next kernel counts on this one having waited for those in front
    return;
  }
  auto begins_at = [&](int w) { return tiles * w / workers; };
  const long long a_begin = begins_at(cta), a_end = begins_at(cta + 1);
  volatile int* aborted = &abort_s;

  // request, head and tile of a tile in the row of all
  auto locate = [&](long long a, int& r, int& kvh, int& t, int& n) {
    int lo = 0, hi = p.R;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)cum[mid] * p.Hkv <= a) lo = mid;
      else hi = mid;
    }
    r = lo;                        // (of requests without tiles at the same place the last one: it has some)
    n = cum[r + 1] - cum[r];
    const int rem = (int)(a - (long long)cum[r] * p.Hkv);
    kvh = rem / n, t = rem % n;
  };

  // ---- this warp's tiles a_begin + warp, + WARPS, ... through its ring. Lane i looks tile `base + i` up and asks for its copies.
  const int mine_n = (int)((a_end - a_begin - warp + WARPS - 1) / WARPS);
  const int boxes = TK / box_rows;                 // 1 or 2
  int looked_up = -32;
  int pg[2] = {-1, -1}, line = 0, head = 0;
  float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
  int issued = 0;
  auto issue = [&](int t) {
    if (t >= mine_n) return;
    issued = t + 1;
    if (t >= looked_up + 32) {
      looked_up = t;
      if (t + lane < mine_n) {
        int r, tile, n, lo, hi, pos0, nrows;
        locate(a_begin + warp + (long long)WARPS * (t + lane), r, head, tile, n);
        span(r, lo, hi, pos0, nrows);
        const int key0 = (lo / TK + tile) * TK;
        const int32_t* table = p.block_table + (size_t)r * p.table_width;
        line = key0 % p.page;
#pragma unroll
        for (int b = 0; b < 2; ++b) {              // the page of each sixteen
          const int key = key0 + 16 * b, slot = key / p.page;
          const int page = key <= hi && slot < p.table_width ? table[slot] : -1;
          const size_t where = (size_t)max(page, 0) * p.Hkv + head;
          // no page: nothing is read there
          const float ks = page >= 0 ? p.k_scale[where] : -1.f, vs = page >= 0 ? p.v_scale[where] : 1.f;
          pg[b] = page;
          const float ev = log2f(vs);
          if (b == 0) sc.x = ks, sc.z = ev;
          else sc.y = ks, sc.w = ev;
        }
      }
    }
    const int s = warp * S::DEPTH + t % S::DEPTH;
    if (lane == t - looked_up) {
      const uint32_t bar = smem_u32(&full_bar[s]), kdst = smem_u32(ring + s * S::STAGE), vdst = kdst + S::OPERAND;
      scale_s[s] = sc;
      // what the warp read from or wrote to this stage is ordered before the copies that overwrite it
      fence_proxy_async();
      mbar_arrive_expect_tx(bar, S::STAGE);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (b >= boxes) break;
        // a page that is not there (-1) is outside the tensor and reads as zeros
        tma_load_4d(kdst + b * box_rows * HD, &k_map, bar, 0, boxes == 1 ? line : 0, head, pg[b]);
        tma_load_4d(vdst + b * box_rows * HD, &v_map, bar, 0, boxes == 1 ? line : 0, head, pg[b]);
      }
    }
    __syncwarp();
  };
  // Everything that is read comes from the kernels in front, the pages among it: a page that this step writes is encoded again.
  gb::pdl_wait();
  for (int t = 0; t < S::DEPTH; ++t) issue(t);

  int t = 0;                       // of this warp's tiles
  for (long long a = a_begin; a < a_end;) {
    // ---- one request's head (or this CTA's part of it): tiles first .. first + count of its n
    int r, kvh, first, n, lo, hi, pos0, nrows;
    locate(a, r, kvh, first, n);
    span(r, lo, hi, pos0, nrows);
    const int count = (int)min((long long)(n - first), a_end - a);
    const int q_begin = p.cu_q[r];

    // the query rows as codes: row lane / 4 (of each eight), hi and lo
    uint32_t qf[MT][HD / 32][4];
    float factor[MT];              // of a row's raw products, times ks: 2^e * scale * log2(e)
    int row_pos[MT], row_start[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int row = mt * 8 + lane / 4;
      const bool there = row < nrows;
      row_pos[mt] = there ? pos0 + row / p.g : -1;
      row_start[mt] = there && p.window > 0 ? max(0, row_pos[mt] + 1 - p.window) : 0;
      const __nv_bfloat16* src = p.q + ((size_t)(q_begin + (there ? row / p.g : 0)) * p.Hq + kvh * p.g + (there ? row % p.g : 0)) * HD + 4 * (lane % 4);
      uint2 raw[HD / 16];
      float largest = 0.f;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        raw[c] = there ? *reinterpret_cast<const uint2*>(src + c * 16) : make_uint2(0u, 0u);
        const float x[4] = {__uint_as_float(raw[c].x << 16), __uint_as_float(raw[c].x & 0xFFFF0000u), __uint_as_float(raw[c].y << 16),
                            __uint_as_float(raw[c].y & 0xFFFF0000u)};
#pragma unroll
        for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(x[e]));
      }
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      const int e2 = f8::scale_exponent(largest);
      const float inv = f8::power_of_two(-e2);
      factor[mt] = f8::power_of_two(e2) * p.scale_log2;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        const float x[4] = {__uint_as_float(raw[c].x << 16) * inv, __uint_as_float(raw[c].x & 0xFFFF0000u) * inv,
                            __uint_as_float(raw[c].y << 16) * inv, __uint_as_float(raw[c].y & 0xFFFF0000u) * inv};
        const uint32_t h = f8::encode4(x[0], x[1], x[2], x[3]);
        const float4 back = f8::decode4(h);
        const int kk = c >> 1, odd = (c & 1) * 2;
        qf[mt][kk][odd] = h;                                       // row i: the code
        qf[mt][kk][odd + 1] = f8::encode4(x[0] - back.x, x[1] - back.y, x[2] - back.z, x[3] - back.w);       // row i + 8: what it leaves
      }
    }

    float o[MT][HD / 8][4], m[MT], l[MT];
    float vref = -200.f;           // log2 of the vs in whose units the sums are
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt] = -INFINITY, l[mt] = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][i][e] = 0.f;
    }

    for (; t < mine_n; ++t) {
      const long long at = a_begin + warp + (long long)WARPS * t - a;           // within this segment
      if (at >= count) break;
      const int s = warp * S::DEPTH + t % S::DEPTH;
      const bool gave_up = __shfl_sync(0xffffffffu, (int)*aborted, 0) != 0;
      if (t >= issued) continue;       // (only after a wait ran out)
      const bool have = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full_bar[s]), (t / S::DEPTH) & 1, gave_up ? DRAIN_LIMIT_NS : WAIT_LIMIT_NS));
      if (!have) {
        if (lane == 0) gb_err::report(ERR_WAIT_FULL);
        *aborted = 1;
        continue;
      }
      if (gave_up) continue;       // what was asked for has landed; nothing more is asked for
      const uint32_t ks_addr = smem_u32(ring + s * S::STAGE), vs_addr = ks_addr + S::OPERAND;
      const float4 scales = scale_s[s];
      const int key0 = (lo / TK + first + (int)at) * TK;
      const bool edge = key0 < lo || key0 + TK - 1 > hi;
      if (edge) {
        // value rows that no query may read are cleared (a weight of zero times a code that is no number would spoil a sum)
        for (int e = lane; e < TK * (HD / 16); e += 32) {
          const int key = e / (HD / 16), c = e % (HD / 16);
          if (key0 + key < lo || key0 + key > hi)
            *reinterpret_cast<uint4*>(ring + s * S::STAGE + S::OPERAND + swizzled<HD>(key, c)) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
      }
      // ---- scores: rows' hi and lo by 32 keys
      float sr[MT][4][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sr[mt][j][e] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // column n of product j is slot 4 (n / 2) + 2 (j & 1) + n % 2 of sixteen j / 2
        const int nn = lane & 7, krow = (j >> 1) * 16 + key_of_slot(4 * (nn >> 1) + 2 * (j & 1) + (nn & 1));
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) {
          uint32_t b[4];
          ldmatrix_x4(b, ks_addr + swizzled<HD>(krow, 4 * h + (lane >> 3)));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma_e4m3(sr[mt][j], qf[mt][2 * h], b[0], b[1]);
            mma_e4m3(sr[mt][j], qf[mt][2 * h + 1], b[2], b[3]);
          }
        }
      }
      // ---- mask, maximum
      const bool full = !edge && scales.x >= 0.f && scales.y >= 0.f && key0 + TK - 1 <= pos0 &&
                        (p.window <= 0 || key0 >= hi + 1 - p.window);
      float sv[MT][8];             // slots (j, e) as 2 j + e, in powers of two
      bool more = false;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float f0 = factor[mt] * scales.x, f1 = factor[mt] * scales.y;
        float mx = m[mt];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = i >> 1, e = i & 1;
          float x = (sr[mt][j][e] + sr[mt][j][e + 2]) * (j < 2 ? f0 : f1);
          if (!full) {
            const int key = key0 + (j >> 1) * 16 + key_of_slot(4 * (lane & 3) + 2 * (j & 1) + e);
            if (key < row_start[mt] || key > row_pos[mt] || (j < 2 ? scales.x : scales.y) < 0.f) x = -INFINITY;
          }
          sv[mt][i] = x;
          mx = fmaxf(mx, x);
        }
        more = more || mx > m[mt];
      }
      // a larger score than any so far (rare after the first tiles), or a larger vs: everything is brought to it
      if (__any_sync(0xffffffffu, more)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float mx = m[mt];
#pragma unroll
          for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sv[mt][i]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float corr = m[mt] == -INFINITY ? 0.f : exp2_fast(m[mt] - mx);
          m[mt] = mx;
          l[mt] *= corr;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][i][e] *= corr;
        }
      }
      const float evm = fmaxf(scales.x >= 0.f ? scales.z : -200.f, scales.y >= 0.f ? scales.w : -200.f);
      if (evm > vref) {
        const float corr = exp2_fast(vref - evm);
        vref = evm;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][i][e] *= corr;
      }
      // ---- weights * 256 * vs / 2^vref as two codes each, the denominator without vs
      uint32_t pf[MT][4];
      // (2^-100 of the largest vs is nothing; and without a page the weights are zeros)
      const float up0 = 8.f + fminf(fmaxf(scales.z - vref, -100.f), 0.f), up1 = 8.f + fminf(fmaxf(scales.w - vref, -100.f), 0.f);
      const float down0 = exp2_fast(-up0), down1 = exp2_fast(-up1);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float base = m[mt] == -INFINITY ? 0.f : -m[mt];
        float w[8], l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = exp2_fast(sv[mt][i] + (base + (i < 4 ? up0 : up1)));
          if (i < 4) l0 += w[i];
          else l1 += w[i];
        }
        l[mt] += l0 * down0 + l1 * down1;
        uint32_t h[4], q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(w[2 * j], w[2 * j + 1], h[j], q[j]);
        pf[mt][0] = h[0] | (h[1] << 16), pf[mt][1] = q[0] | (q[1] << 16);
        pf[mt][2] = h[2] | (h[3] << 16), pf[mt][3] = q[2] | (q[3] << 16);
      }
      // ---- sums of the values
      const int vrow = key_of_slot(lane);          // slot lane of 32 (bit 4 stays)
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t b[4];
        ldmatrix_trans_bytes(b, vs_addr + swizzled<HD>(vrow, c));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma_e4m3(o[mt][2 * c], pf[mt], b[0], b[2]);
          mma_e4m3(o[mt][2 * c + 1], pf[mt], b[1], b[3]);
        }
      }
      __syncwarp();                // every lane is done with the stage before it is filled again
      issue(t + S::DEPTH);
    }
    // ---- the warps' sums are merged in shared memory, CW channels at a time
    const float unit = exp2_fast(vref - 8.f);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 1);
      l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 2);
      if (lane % 4 == 0) ml_s[warp][mt * 8 + lane / 4] = make_float2(m[mt], l[mt]);
    }
    const bool whole = first == 0 && count == n;
    const long long seg0 = a - first;              // the segment's first tile in the row of all
    float* my_part = partials + ((size_t)cta * 2 + (a == a_begin ? 0 : 1)) * (MAX_ROWS * RS);
    constexpr int LANES = THREADS / ROWS;          // threads of a row: 16 or 8
    const int row = threadIdx.x / LANES, sub = threadIdx.x % LANES;
    __nv_bfloat16* const dst = p.out + ((size_t)(q_begin + (row < nrows ? row / p.g : 0)) * p.Hq + kvh * p.g + (row < nrows ? row % p.g : 0)) * HD;
#pragma unroll
    for (int pass = 0; pass < S::PASSES; ++pass) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float* to = red + (warp * ROWS + mt * 8 + lane / 4) * CW + (lane % 4) * 2;
#pragma unroll
        for (int i = 0; i < CW / 8; ++i) {
          const float* x = o[mt][pass * (CW / 8) + i];
          *reinterpret_cast<float2*>(to + i * 8) = make_float2((x[0] + x[2] * 0.03125f) * unit, (x[1] + x[3] * 0.03125f) * unit);
        }
      }
      __syncthreads();
      float f[WARPS], mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, ml_s[w][row].x);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float2 x = ml_s[w][row];
        f[w] = x.x == -INFINITY ? 0.f : exp2_fast(x.x - mm);
        ll += f[w] > 0.f ? f[w] * x.y : 0.f;
      }
      if (row < nrows) {
        const float inv = ll > 0.f ? 1.0f / ll : 0.f;
#pragma unroll
        for (int c = 2 * sub; c < CW; c += 2 * LANES) {
          float2 v = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            const float2 x = *reinterpret_cast<const float2*>(red + (w * ROWS + row) * CW + c);
            if (f[w] > 0.f) v.x += f[w] * x.x, v.y += f[w] * x.y;          // (a warp without a key has nothing)
          }
          if (whole) gb::store_pair(dst + pass * CW + c, v.x * inv, v.y * inv);
          else __stcg(reinterpret_cast<float2*>(my_part + row * RS + pass * CW + c), v);
        }
        if (!whole && pass == 0 && sub == 0) __stcg(reinterpret_cast<float2*>(my_part + row * RS + HD), make_float2(mm, ll));
      }
      __syncthreads();             // the buffer is free for the next pass, or the next segment
    }
    if (!whole) {
      // ---- several CTAs: who counts the last arrival adds the parts up, in the CTAs' order
      int w0 = (int)(seg0 * workers / tiles), w1 = (int)((seg0 + n - 1) * workers / tiles);
      while (w0 + 1 < workers && begins_at(w0 + 1) <= seg0) ++w0;
      while (w0 > 0 && begins_at(w0) > seg0) --w0;
      while (w1 + 1 < workers && begins_at(w1 + 1) <= seg0 + n - 1) ++w1;
      while (w1 > 0 && begins_at(w1) > seg0 + n - 1) --w1;
      if (threadIdx.x == 0) {      // (behind the barrier in front: all have written their part)
        __threadfence();
        int* counter = counters + (size_t)r * p.Hkv + kvh;
        last_s = atomicAdd(counter, 1) == w1 - w0;
        if (last_s) *counter = 0;                  // as the next launch expects it
        __threadfence();
      }
      __syncthreads();
      if (last_s) {
        auto part_of = [&](int w) {      // only the first of them may hold another segment's end in front of its part
          return partials + ((size_t)w * 2 + (w == w0 && begins_at(w0) < seg0 ? 1 : 0)) * (MAX_ROWS * RS);
        };
        if (row < nrows) {
          constexpr int PER = HD / LANES / 2;
          float mm = -INFINITY, ll = 0.f;
          float2 v[PER];
          for (int w = w0; w <= w1; ++w) mm = fmaxf(mm, __ldcg(part_of(w) + row * RS + HD));
#pragma unroll
          for (int i = 0; i < PER; ++i) v[i] = make_float2(0.f, 0.f);
#pragma unroll 4
          for (int w = w0; w <= w1; ++w) {
            const float* part = part_of(w) + row * RS;
            const float2 x = __ldcg(reinterpret_cast<const float2*>(part + HD));
            const float f = x.x == -INFINITY ? 0.f : exp2_fast(x.x - mm);
            ll += f > 0.f ? f * x.y : 0.f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const float2 y = __ldcg(reinterpret_cast<const float2*>(part + 2 * (sub + LANES * i)));
              if (f > 0.f) v[i].x += f * y.x, v[i].y += f * y.y;
            }
          }
          const float inv = ll > 0.f ? 1.0f / ll : 0.f;
#pragma unroll
          for (int i = 0; i < PER; ++i) gb::store_pair(dst + 2 * (sub + LANES * i), v[i].x * inv, v[i].y * inv);
        }
      }
      __syncthreads();             // the flag is free for the next segment
    }
    a += count;
  }
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

// Pools [pages][heads][page][hd] of bytes through boxes [1][1][min(page, 32)][hd], swizzled over the rows' width.
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
  cuuint32_t box[4] = {(cuuint32_t)hd, (cuuint32_t)(page < TK ? page : TK), 1, 1};
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

constexpr int CTAS = 2;               // per SM
constexpr int MAX_REQUESTS = 1024;    // their tiles' sums lie in shared memory

template <int HD, int MT>
int launch(const Params& p, const CUtensorMap& km, const CUtensorMap& vm, int grid, int min_tiles, void* parts, void* counters, cudaStream_t stream) {
  auto kernel = attention_f8_decode_kernel<HD, MT>;
  using S = Shape<HD, MT>;
  constexpr int MOST = 1024 + S::RING + S::MERGE + (MAX_REQUESTS + 1) * 4;
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "attention_f8_decode: %s", cudaGetErrorString(e));
    configured.done();
  }
  const size_t smem = 1024 + S::RING + S::MERGE + (size_t)(p.R + 1) * 4;
  return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3((unsigned)grid), dim3(THREADS), smem, stream, dim3(1), km, vm, p, p.page < TK ? p.page : TK,
                                             min_tiles, (float*)parts, (int*)counters), "attention_f8_decode");
}

}  // namespace

// Whether the kernel takes this shape: heads of 64 or 128, pages of 16, 32, 64 or 128 keys, up to sixteen query heads a group, up to 1,024 requests.
GB_EXPORT int gb_f8_attention_decode_takes(int hd, int page, int g, int R) {
  return (hd == 64 || hd == 128) && page >= 16 && page <= 128 && (page & (page - 1)) == 0 && g <= 16 && R <= MAX_REQUESTS && tc_host::encode_fn() != nullptr;
}
// Rows (new tokens times heads of a group) up to which a request is its.
GB_EXPORT int gb_f8_attention_decode_rows(int g) { return attn8::decode_rows(g); }
// Bytes of the parts that CTAs leave to one another (no need to clear them) and of the counters (zero before the first launch; every
// launch leaves them zero).
GB_EXPORT long long gb_f8_attention_decode_scratch(int R, int Hkv, int hd, long long* counters) {
  *counters = ((long long)R * Hkv * 4 + 255) / 256 * 256;
  return (long long)tc_host::sm_count() * CTAS * 2 * MAX_ROWS * (hd + 2) * 4;
}

GB_EXPORT int gb_f8_attention_decode(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale, const void* table,
                                     int table_width, const void* cu_q, const void* kv_lens, void* out, int R, long long pages, int Hq, int Hkv, int hd,
                                     float scale, int window, int page, int max_kv_len, void* parts, void* counters, void* stream) {
  const int g = Hq / Hkv;
  if (R <= 0 || Hkv <= 0 || Hq % Hkv || !gb_f8_attention_decode_takes(hd, page, g, R) || (uintptr_t)q % 8 || (uintptr_t)out % 4 || (uintptr_t)k_pool % 16 ||
      (uintptr_t)v_pool % 16)
    return gb::fail(GB_BAD_ARGUMENT, "attention_f8_decode: %d requests, heads %d / %d of %d, pages of %d", R, Hq, Hkv, hd, page);
  Params p{(const __nv_bfloat16*)q, (const float*)k_scale, (const float*)v_scale, (__nv_bfloat16*)out, (const int32_t*)table, (const int32_t*)cu_q,
           (const int32_t*)kv_lens, table_width, R, Hq, Hkv, g, window, page, attn8::decode_rows(g), scale * 1.4426950408889634f};
  CUtensorMap km, vm;
  int rc = pool_map(k_pool, page, Hkv, pages, hd, &km);
  if (rc) return rc;
  rc = pool_map(v_pool, page, Hkv, pages, hd, &vm);
  if (rc) return rc;
  const int reach = window > 0 && window + 2 * TK < max_kv_len ? window + 2 * TK : max_kv_len;
  // Four tiles a warp at least: a shorter stretch costs more in parts to merge than it saves (500 keys, 8 heads: 10.7 us from 4 tiles a CTA
  // on, 8.6 from 16, 15.1 from 32).
  const int min_tiles = 16;
  const long long most = (long long)R * Hkv * ((reach + TK - 1) / TK + 1) / min_tiles + 1;
  const int room = tc_host::sm_count() * CTAS, grid = (int)(most < room ? most : room);
  const cudaStream_t st = (cudaStream_t)stream;
  if (hd == 64) return g <= 8 ? launch<64, 1>(p, km, vm, grid, min_tiles, parts, counters, st) : launch<64, 2>(p, km, vm, grid, min_tiles, parts, counters, st);
  return g <= 8 ? launch<128, 1>(p, km, vm, grid, min_tiles, parts, counters, st) : launch<128, 2>(p, km, vm, grid, min_tiles, parts, counters, st);
}

GB_EXPORT int gb_f8_attention_decode_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_f8_attention_decode_set_error_sink(void* host_word) { return gb_err::set_sink((int*)host_word); }
