// The 8-bit path's elementwise kernels and its plain attention: tokens' rows into codes, a step's keys and values into
// pages of codes with the rotation on the way, and attention over such pages for the shapes that the tensor-core kernels
// (attention_float8_decode.cu, attention_float8_tile.cu) do not take.
//
// The reference keeps its cache in 32 bits (garuda/src/cache/mod.rs:221-241) and its weights in GGUF's block formats; the formulas
// around the codes are its own: rotation garuda/src/simd/mod.rs:196-206, attention garuda/src/llama/mod.rs:793-818, window
// garuda/src/cache/mod.rs:333-338.
#include "float8.cuh"

namespace {

using namespace f8;

// ------------------------------------------------------------------ tokens into codes
// a [M, K] -> codes [M, pitch] and, per token and 128 channels, the exponent byte of the scale (e + 127), those of four blocks in a
// word: [blocks / 4 rounded up][M][4]. Sixteen lanes take a block, eight
// channels each, so that a warp reads two blocks of a row (512 bytes of bfloat16) in one instruction; a block's largest
// magnitude takes four shuffles. Bound by memory; what is read is kept in registers, so nothing is read twice.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* src, int have, float (&x)[8]) {
  if (WIDE && have >= 8) {
    if (sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(src);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    } else {
      const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < have ? gb::to_float(src[i]) : 0.f;
  }
}

// GATED: rows are [gate | up], K channels each, and silu(gate) * up is what becomes codes, from 32 bits at once.
template <typename T, bool WIDE, bool GATED>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ a, long long lda, int M, int K, uint8_t* __restrict__ codes, int pitch,
                     uint8_t* __restrict__ scales) {
  gb::pdl_launch_dependents();
  const uint32_t kb = (uint32_t)(K + BLOCK - 1) / BLOCK, all = (uint32_t)M * kb;
  const uint32_t block = blockIdx.x * 16 + (threadIdx.x >> 4);       // of all rows'; the host has seen that they fit 31 bits
  if (block - (threadIdx.x & 16 ? 1 : 0) >= all) return;             // the warp's first block lies behind the last
  const bool mine = block < all;
  const int row = mine ? (int)(block / kb) : 0, b = mine ? (int)(block - (uint32_t)row * kb) : 0;
  gb::pdl_wait();
  const int k = b * BLOCK + (threadIdx.x & 15) * 8;
  float x[8];
  load8<T, WIDE>(a + row * lda + k, mine ? K - k : 0, x);
  if (GATED) {
    float up[8];
    load8<T, WIDE>(a + row * lda + K + k, mine ? K - k : 0, up);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] / (1.0f + expf(-x[i])) * up[i];
  }
  float largest = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  const int e = scale_exponent(largest);
  const float inv = power_of_two(-e);
  if (!mine) return;
  if (k < pitch) {       // pitch is a multiple of 16: whole eights
    uint2 c;
    c.x = encode4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    c.y = encode4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    *reinterpret_cast<uint2*>(codes + (size_t)row * pitch + k) = c;
  }
  if ((threadIdx.x & 15) == 0) scales[((size_t)(b >> 2) * M + row) * 4 + (b & 3)] = (uint8_t)(e + 127);
}

// ------------------------------------------------------------------ weights into codes
// One block of threads per 128 x 128 of w [N, K]; a load-time kernel. It does not let the kernel behind it start early: the
// products fetch weights before they wait for the kernel in front of them.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_weight_kernel(const T* __restrict__ w, long long ldw, int N, int K, uint8_t* __restrict__ codes, long long pitch, float* __restrict__ scales) {
  __shared__ float part[8];
  const int k0 = blockIdx.x * BLOCK, n0 = blockIdx.y * BLOCK, k = k0 + (threadIdx.x & 127);
  float largest = 0.f;
  for (int n = n0 + (threadIdx.x >> 7); n < min(N, n0 + BLOCK); n += 2)
    if (k < K) largest = fmaxf(largest, fabsf(gb::to_float(w[n * ldw + k])));
  largest = gb::warp_max(largest);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = largest;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = fmaxf(largest, part[i]);
  const int e = scale_exponent(largest);
  const float inv = power_of_two(-e);
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = power_of_two(e);
  for (int n = n0 + (threadIdx.x >> 7); n < min(N, n0 + BLOCK); n += 2)
    if (k < pitch) codes[n * pitch + k] = (uint8_t)encode2(k < K ? gb::to_float(w[n * ldw + k]) * inv : 0.f, 0.f);
}

// ------------------------------------------------------------------ keys and values into pages of codes
// One block per (page that the step writes, key/value head). With h rows of the page held before:
//   s' = scale(largest |new|), or the larger of that and s where h > 0;  old codes <- enc(code * s / s');  new ones enc(x / s')
// Every page that a step writes belongs to one request, and of these only the first holds old rows, so no two blocks touch a page of
// a head. A request with q new tokens writes at most floor(q / page) + 2 pages; its blocks start at floor(cu_q / page) + 2 r, which
// every block inverts by bisection: no plan from the host, and a grid that depends on the sizes alone.
template <typename T>
__device__ __forceinline__ float2 load2(const T* p);
template <>
__device__ __forceinline__ float2 load2<float>(const float* p) { return *reinterpret_cast<const float2*>(p); }
template <>
__device__ __forceinline__ float2 load2<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
}

// Four channels of a head: two pairs, each rotated. Half layout: channels c, c + 1 and their partners c + half, c + half + 1, c = 2 j;
// interleaved: the pairs (4 j, 4 j + 1), (4 j + 2, 4 j + 3). Products and sums are rounded one by one (no fused multiply-add), so that a
// code does not depend on which of two products a compiler fuses.
struct Four {
  float2 a, b;       // half: first halves, second halves; interleaved (and not rotated): channels 4 j, 4 j + 1 and 4 j + 2, 4 j + 3
};
template <typename T>
__device__ __forceinline__ Four load_four(const T* x, int j, int half, bool split) {
  Four f;
  f.a = load2(x + (split ? 2 * j : 4 * j));
  f.b = load2(x + (split ? half + 2 * j : 4 * j + 2));
  return f;
}
// (t: cos, sin of pair 2 j, cos, sin of pair 2 j + 1)
__device__ __forceinline__ void rotate(Four& f, float4 t, bool split) {
  float& x0 = f.a.x;
  float& y0 = split ? f.b.x : f.a.y;
  float& x1 = split ? f.a.y : f.b.x;
  float& y1 = f.b.y;
  const float u0 = __fsub_rn(__fmul_rn(x0, t.x), __fmul_rn(y0, t.y)), v0 = __fadd_rn(__fmul_rn(x0, t.y), __fmul_rn(y0, t.x));
  const float u1 = __fsub_rn(__fmul_rn(x1, t.z), __fmul_rn(y1, t.w)), v1 = __fadd_rn(__fmul_rn(x1, t.w), __fmul_rn(y1, t.z));
  x0 = u0, y0 = v0, x1 = u1, y1 = v1;
}
__device__ __forceinline__ float largest_of(const Four& f) {
  return fmaxf(fmaxf(fabsf(f.a.x), fabsf(f.a.y)), fmaxf(fabsf(f.b.x), fabsf(f.b.y)));
}
__device__ __forceinline__ void store_codes(uint8_t* row, const Four& f, float inv, int j, int half, bool split) {
  const uint16_t a = encode2(f.a.x * inv, f.a.y * inv), b = encode2(f.b.x * inv, f.b.y * inv);
  if (split) {
    *reinterpret_cast<uint16_t*>(row + 2 * j) = a;
    *reinterpret_cast<uint16_t*>(row + half + 2 * j) = b;
  } else {
    *reinterpret_cast<uint32_t*>(row + 4 * j) = (uint32_t)a | ((uint32_t)b << 16);
  }
}

struct Append {
  const void* qkv;
  long long qkv_stride;
  void* q_out;
  uint8_t *k_pool, *v_pool;
  float *k_scale, *v_scale;
  const int32_t *cu_q, *kv_lens, *table;
  int table_width, T, R, Hq, Hkv, hd, page;
  const float* cos_sin;       // [T, hd / 2, 2] or null
  bool interleaved;
};

constexpr int APPEND_THREADS = 256;
constexpr int KEPT = 4;         // rows of keys and of values that a thread keeps in registers between their maximum and their codes
constexpr int QUERIES = 4;      // heads of a piece of queries

// A piece of work is one head of a page's keys and values, or QUERIES heads of its tokens' queries (they wait for no maximum); WARPS of a
// block have one. Lanes lie along a row (four channels each; short rows share a warp), a piece's warps take the rows in turn. KEEP: a
// thread's first KEPT rows are read once, and with eight warps these are all (page * head size <= 4,096: 32 keys of 128 channels; else,
// and what a single warp has beyond them, is read twice).
template <typename TI, typename TO, bool KEEP, int WARPS>
__global__ void __launch_bounds__(APPEND_THREADS, WARPS == 1 ? 2 : 4) append_kernel(const Append p) {
  gb::pdl_launch_dependents();
  __shared__ float part[2][WARPS];
  const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5, thread = WARPS == 1 ? lane : threadIdx.x;       // of the piece
  const int piece = WARPS == 1 ? blockIdx.y * (APPEND_THREADS / 32) + (threadIdx.x >> 5) : blockIdx.y;
  if (piece >= p.Hkv + (p.Hq + QUERIES - 1) / QUERIES) return;
  // the request of this page: the last one that starts at or before it, found by 32 lanes at a time
  int lo = 0;
  const int slot = blockIdx.x;
  for (int left = p.R; left > 1;) {
    const int apart = (left + 31) / 32, i = lo + lane * apart;
    const bool before = lane * apart < left && p.cu_q[i] / p.page + 2 * i <= slot;
    const int skip = max(__popc(__ballot_sync(0xffffffffu, before)) - 1, 0) * apart;
    lo += skip, left = min(apart, left - skip);
  }
  const int r = lo, begin = p.cu_q[r], q_len = p.cu_q[r + 1] - begin;
  const int pos0 = p.kv_lens[r] - q_len;
  const int page_index = pos0 / p.page + (slot - (begin / p.page + 2 * r));
  const int first = max(pos0, page_index * p.page), last = min(p.kv_lens[r], (page_index + 1) * p.page);
  if (q_len <= 0 || first >= last) return;
  const int at = page_index < p.table_width ? p.table[(size_t)r * p.table_width + page_index] : -1;       // (no page: the queries are written all the same)
  const int n = last - first, held = first - page_index * p.page;
  const int tok0 = begin + first - pos0;

  const int half = p.hd / 2, fours = p.hd / 4;
  const bool rotated = p.cos_sin != nullptr, split = rotated && !p.interleaved;
  // this thread's place: row `row0` of every `step`, channels 4 j0 (and, in rows of more than 128, 4 (j0 + 32))
  const int shared = fours == 16 ? 2 : fours == 8 ? 4 : fours == 4 ? 8 : 1;          // rows of a warp
  const int row0 = warp * shared + (shared > 1 ? lane / fours : 0), step = WARPS * shared;
  const int j0 = shared > 1 ? lane % fours : lane;
  const TI* rows = reinterpret_cast<const TI*>(p.qkv) + tok0 * p.qkv_stride;
  const float* angles = p.cos_sin + (size_t)tok0 * p.hd;
  if (piece >= p.Hkv) {
    const int h0 = (piece - p.Hkv) * QUERIES, heads = min(QUERIES, p.Hq - h0);
    TO* const q_out = reinterpret_cast<TO*>(p.q_out) + ((size_t)tok0 * p.Hq + h0) * p.hd;
    gb::pdl_wait();
#pragma unroll 1
    for (int t = row0; t < n; t += step) {
      for (int j = j0; j < fours; j += 32) {
        float4 turn{};          // the heads' one rotation
        if (rotated) turn = *reinterpret_cast<const float4*>(angles + (size_t)t * p.hd + 4 * j);
        Four q[QUERIES];
#pragma unroll
        for (int h = 0; h < QUERIES; ++h)
          if (h < heads) q[h] = load_four(rows + t * p.qkv_stride + (size_t)(h0 + h) * p.hd, j, half, split);
#pragma unroll
        for (int h = 0; h < QUERIES; ++h) {
          if (h >= heads) break;
          if (rotated) rotate(q[h], turn, split);
          TO* to = q_out + ((size_t)t * p.Hq + h) * p.hd;
          gb::store_pair(to + (split ? 2 * j : 4 * j), q[h].a.x, q[h].a.y);
          gb::store_pair(to + (split ? half + 2 * j : 4 * j + 2), q[h].b.x, q[h].b.y);
        }
      }
    }
    return;
  }
  const int kvh = piece;
  if (at < 0) return;
  const TI* keys = rows + (size_t)(p.Hq + kvh) * p.hd;
  const TI* values = keys + (size_t)p.Hkv * p.hd;
  auto key = [&](int t, int j) {
    Four k = load_four(keys + t * p.qkv_stride, j, half, split);
    if (rotated) rotate(k, *reinterpret_cast<const float4*>(angles + (size_t)t * p.hd + 4 * j), split);
    return k;
  };
  auto value = [&](int t, int j) { return load_four(values + t * p.qkv_stride, j, half, false); };
  const size_t where = (size_t)at * p.Hkv + kvh;
  gb::pdl_wait();
  const float old_k = held ? p.k_scale[where] : 0.f, old_v = held ? p.v_scale[where] : 0.f;
  float mk = 0.f, mv = 0.f;
  Four ks[KEEP ? KEPT : 1], vs[KEEP ? KEPT : 1];
  if (KEEP) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int t = row0 + i * step;
      if (t < n && j0 < fours) {
        ks[i] = key(t, j0), vs[i] = value(t, j0);
        mk = fmaxf(mk, largest_of(ks[i])), mv = fmaxf(mv, largest_of(vs[i]));
      }
    }
  }
  const int again = KEEP ? row0 + KEPT * step : row0;          // the first row that is read twice
  if (!KEEP || WARPS == 1) {
    for (int t = again; t < n; t += step)
      for (int j = j0; j < fours; j += 32) mk = fmaxf(mk, largest_of(key(t, j))), mv = fmaxf(mv, largest_of(value(t, j)));
  }
  mk = gb::warp_max(mk), mv = gb::warp_max(mv);
  if (WARPS > 1) {
    if (lane == 0) part[0][warp] = mk, part[1][warp] = mv;
    __syncthreads();
    mk = part[0][0], mv = part[1][0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) mk = fmaxf(mk, part[0][w]), mv = fmaxf(mv, part[1][w]);
  } else {
    __syncwarp();          // (every lane has read the old scales)
  }
  const float sk = fmaxf(old_k, power_of_two(scale_exponent(mk))), sv = fmaxf(old_v, power_of_two(scale_exponent(mv)));
  if (thread == 0) p.k_scale[where] = sk, p.v_scale[where] = sv;       // (every thread has read the old ones)
  uint8_t* kp = p.k_pool + where * p.page * p.hd;
  uint8_t* vp = p.v_pool + where * p.page * p.hd;
  // the scale has grown: the rows that were there are encoded again
  for (int which = 0; which < 2; ++which) {
    const float s = which ? sv : sk, old = which ? old_v : old_k;
    if (held == 0 || s == old) continue;
    uint32_t* codes = reinterpret_cast<uint32_t*>(which ? vp : kp);
    const float factor = old / s;
#pragma unroll 4
    for (int i = thread; i < held * fours; i += 32 * WARPS) {
      const float4 x = decode4(codes[i]);
      codes[i] = encode4(x.x * factor, x.y * factor, x.z * factor, x.w * factor);
    }
  }
  const float ik = 1.0f / sk, iv = 1.0f / sv;        // powers of two: exact
  if (KEEP) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int t = row0 + i * step;
      if (t < n && j0 < fours) {
        store_codes(kp + (size_t)(held + t) * p.hd, ks[i], ik, j0, half, split);
        store_codes(vp + (size_t)(held + t) * p.hd, vs[i], iv, j0, half, false);
      }
    }
  }
  if (!KEEP || WARPS == 1) {
    for (int t = again; t < n; t += step)
      for (int j = j0; j < fours; j += 32) {
        store_codes(kp + (size_t)(held + t) * p.hd, key(t, j), ik, j, half, split);
        store_codes(vp + (size_t)(held + t) * p.hd, value(t, j), iv, j, half, false);
      }
  }
}

// ------------------------------------------------------------------ attention, any shape
// A warp per (token, query head): its lanes share out the channels, four at a time, and walk the keys with a running maximum and
// denominator in 32 bits. For head sizes, pages, groups and types that the tensor-core kernels do not take.
struct AttentionSimple {
  const void* q;
  const uint8_t *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  const int32_t *table, *cu_q, *kv_lens;
  void* out;
  int table_width, T, R, Hq, Hkv, hd, page, window;
  float scale_log2;
};

constexpr int MAX_HD = 256;

template <typename T>
__global__ void __launch_bounds__(128) attention_f8_simple_kernel(const AttentionSimple p) {
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (long long)p.T * p.Hq) return;
  const int t = (int)(row / p.Hq), h = (int)(row % p.Hq), kvh = h / (p.Hq / p.Hkv);
  int lo = 0, hi = p.R;          // the token's request: the last one that starts at or before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int r = lo, pos = p.kv_lens[r] - (p.cu_q[r + 1] - t);
  const int start = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  const int32_t* table = p.table + (size_t)r * p.table_width;
  const T* q = reinterpret_cast<const T*>(p.q) + (size_t)row * p.hd;
  constexpr int PER = MAX_HD / 128;
  float qv[PER][4], o[PER][4];
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 128 * i + 4 * lane + e;
      const float x = c < p.hd ? gb::to_float(q[c]) : 0.f;
      qv[i][e] = x + (x - x);      // (NaN for an infinity: a softmax of infinite scores is no number)
      o[i][e] = 0.f;
    }
  float m = -INFINITY, l = 0.f;
  for (int key = start; key <= pos;) {
    const int slot = key / p.page;
    if (slot >= p.table_width) break;
    const int page = table[slot], line = key % p.page;
    const int end = min(p.page, line + pos + 1 - key);
    if (page < 0) {                      // given back: nothing there
      key += end - line;
      continue;
    }
    const size_t where = (size_t)page * p.Hkv + kvh;
    const float ks = p.k_scale[where] * p.scale_log2, vs = p.v_scale[where];
    const uint8_t* kp = p.k_pool + where * p.page * p.hd;
    const uint8_t* vp = p.v_pool + where * p.page * p.hd;
    for (int j = line; j < end; ++j, ++key) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = 128 * i + 4 * lane;
        if (c < p.hd) {
          const float4 k = decode4(*reinterpret_cast<const uint32_t*>(kp + (size_t)j * p.hd + c));
          s += (qv[i][0] * k.x + qv[i][1] * k.y) + (qv[i][2] * k.z + qv[i][3] * k.w);
        }
      }
      s = gb::warp_sum(s) * ks;
      const float m_new = fmaxf(m, s);
      // (a score that is no number stays one)
      const float corr = m == m_new ? 1.f : exp2f(m - m_new), w = m_new == -INFINITY ? (s == s ? 0.f : s) : exp2f(s - m_new);
      m = m_new;
      l = l * corr + w;
      const float wv = w * vs;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = 128 * i + 4 * lane;
        if (c < p.hd) {
          const float4 v = decode4(*reinterpret_cast<const uint32_t*>(vp + (size_t)j * p.hd + c));
          o[i][0] = o[i][0] * corr + wv * v.x, o[i][1] = o[i][1] * corr + wv * v.y;
          o[i][2] = o[i][2] * corr + wv * v.z, o[i][3] = o[i][3] * corr + wv * v.w;
        }
      }
    }
  }
  const float inv = l > 0.f ? 1.0f / l : (l == l ? 0.f : l);         // no key: zeros
  T* out = reinterpret_cast<T*>(p.out) + (size_t)row * p.hd;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = 128 * i + 4 * lane;
    if (c < p.hd) {
      gb::store_pair(out + c, o[i][0] * inv, o[i][1] * inv);
      gb::store_pair(out + c + 2, o[i][2] * inv, o[i][3] * inv);
    }
  }
}

}  // namespace

GB_DEFINE_LAST_ERROR()

// a [M, K] (rows lda apart; gated: [M, 2 K]) -> codes [M, pitch] (pitch a multiple of 16, at least K; the rest zeros) and scales
// [ceil(K / 512)][M][4] as exponent bytes.
int gb_f8_quantize_rows(const void* a, int tag, long long lda, int gated, int M, int K, void* codes, int pitch, void* scales, cudaStream_t stream) {
  if (M < 0 || K <= 0 || pitch < K || pitch % 16 || (uintptr_t)codes % 16) return gb::fail(GB_BAD_ARGUMENT, "quantize_rows: %d x %d, pitch %d", M, K, pitch);
  if (M == 0) return GB_OK;
  const long long blocks = (long long)M * ((K + f8::BLOCK - 1) / f8::BLOCK);
  const long long grid = (blocks * 16 + 255) / 256;
  if (blocks > 0x7fffffff) return gb::fail(GB_UNSUPPORTED, "quantize_rows: %lld blocks", blocks);
  return GB_DISPATCH_DTYPE(tag, T, [&]() -> int {
    const bool wide = (uintptr_t)a % 16 == 0 && lda * (long long)sizeof(T) % 16 == 0 && (!gated || K * (long long)sizeof(T) % 16 == 0);
    auto* kernel = gated ? (wide ? quantize_rows_kernel<T, true, true> : quantize_rows_kernel<T, false, true>)
                         : (wide ? quantize_rows_kernel<T, true, false> : quantize_rows_kernel<T, false, false>);
    return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3((unsigned)grid), dim3(256), 0, stream, dim3(1), (const T*)a, lda, M, K,
                                               (uint8_t*)codes, pitch, (uint8_t*)scales), "quantize_rows");
  });
}

// w [N, K] (rows ldw apart) -> codes [N, pitch] (pitch a multiple of 16, less than 128 behind K; the rest zeros) and scales
// [ceil(N / 128)][ceil(K / 128)].
GB_EXPORT int gb_f8_quantize_weight(const void* w, int tag, long long ldw, int N, int K, void* codes, long long pitch, void* scales, void* stream) {
  const int kb = (K + f8::BLOCK - 1) / f8::BLOCK, nb = (N + f8::BLOCK - 1) / f8::BLOCK;
  if (N <= 0 || K <= 0 || pitch < K || pitch % 16 || pitch > (long long)kb * f8::BLOCK || nb > 65535)
    return gb::fail(GB_BAD_ARGUMENT, "quantize_weight: %d x %d, pitch %lld", N, K, pitch);
  return GB_DISPATCH_DTYPE(tag, T, [&]() -> int {
    quantize_weight_kernel<T><<<dim3(kb, nb), 256, 0, (cudaStream_t)stream>>>((const T*)w, ldw, N, K, (uint8_t*)codes, pitch, (float*)scales);
    return gb::check_launch("quantize_weight");
  });
}

GB_EXPORT int gb_f8_append(const void* qkv, int tag, long long qkv_stride, void* q_out, int q_tag, void* k_pool, void* v_pool, void* k_scale,
                           void* v_scale, const void* cu_q, const void* kv_lens, const void* table, int table_width, int T, int R, int Hq,
                           int Hkv, int hd, const void* cos_sin, int interleaved, int page, void* stream) {
  if (T < 0 || R <= 0 || Hkv <= 0 || Hq % Hkv || hd % 16 || page <= 0 || Hq > 65535)
    return gb::fail(GB_BAD_ARGUMENT, "f8_append: %d tokens, %d requests, heads %d / %d of %d, pages of %d", T, R, Hq, Hkv, hd, page);
  if (T == 0) return GB_OK;
  Append p{qkv, qkv_stride, q_out, (uint8_t*)k_pool, (uint8_t*)v_pool, (float*)k_scale, (float*)v_scale, (const int32_t*)cu_q,
           (const int32_t*)kv_lens, (const int32_t*)table, table_width, T, R, Hq, Hkv, hd, page, (const float*)cos_sin, interleaved != 0};
  const long long slots = (long long)T / page + 2LL * R;
  if (slots > 0x7fffffff) return gb::fail(GB_UNSUPPORTED, "f8_append: %lld pages", slots);
  return GB_DISPATCH_DTYPE(tag, TI, [&]() -> int {
    return GB_DISPATCH_DTYPE(q_tag, TO, [&]() -> int {
      // Single tokens leave a page one row: a warp a piece (64 tokens of 32 + 8 heads of 128: 2.3 us; eight warps, seven of them idle, 7.6).
      // Else eight (2,047 tokens: 17 us).
      const int pieces = Hkv + (Hq + QUERIES - 1) / QUERIES, fours = hd / 4, shared = fours == 16 ? 2 : fours == 8 ? 4 : fours == 4 ? 8 : 1;
      const bool few = T <= R, fits = hd <= 128 && page <= KEPT * (APPEND_THREADS / 32) * shared;
      auto* kernel = few ? (hd <= 128 ? append_kernel<TI, TO, true, 1> : append_kernel<TI, TO, false, 1>)
                         : (fits ? append_kernel<TI, TO, true, APPEND_THREADS / 32> : append_kernel<TI, TO, false, APPEND_THREADS / 32>);
      const dim3 grid((unsigned)slots, few ? (unsigned)(pieces + APPEND_THREADS / 32 - 1) / (APPEND_THREADS / 32) : (unsigned)pieces);
      return gb::check_pdl_launch(gb::launch_pdl(kernel, grid, dim3(APPEND_THREADS), 0, (cudaStream_t)stream, dim3(1), p),
                                  "f8_append");
    });
  });
}

GB_EXPORT int gb_f8_attention_simple(const void* q, int tag, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                                     const void* table, int table_width, const void* cu_q, const void* kv_lens, void* out, int T, int R,
                                     int Hq, int Hkv, int hd, float scale, int window, int page, void* stream) {
  if (T < 0 || R <= 0 || Hkv <= 0 || Hq % Hkv || hd % 16 || hd > MAX_HD || page <= 0)
    return gb::fail(GB_BAD_ARGUMENT, "f8_attention: %d tokens, %d requests, heads %d / %d of %d, pages of %d", T, R, Hq, Hkv, hd, page);
  if (T == 0) return GB_OK;
  AttentionSimple p{q, (const uint8_t*)k_pool, (const uint8_t*)v_pool, (const float*)k_scale, (const float*)v_scale, (const int32_t*)table,
                    (const int32_t*)cu_q, (const int32_t*)kv_lens, out, table_width, T, R, Hq, Hkv, hd, page, window,
                    scale * 1.4426950408889634f};
  const long long grid = ((long long)T * Hq + 3) / 4;
  if (grid > 0x7fffffff) return gb::fail(GB_UNSUPPORTED, "f8_attention: %lld rows", (long long)T * Hq);
  return GB_DISPATCH_DTYPE(tag, TT, [&]() -> int {
    return gb::check_pdl_launch(gb::launch_pdl(attention_f8_simple_kernel<TT>, dim3((unsigned)grid), dim3(128), 0, (cudaStream_t)stream, dim3(1), p),
                                "f8_attention");
  });
}
