// Attention of drafted trees over the paged cache in 32-bit arithmetic throughout: the true 32-bit path, and bfloat16 where the kernel on
// the tensor cores does not apply (head sizes other than 64 and 128, pages of other sizes). The same formula, see attention_tree_tcgen05.cu.
//
// Bound by the multiply-adds (32-bit ones run on the ordinary pipes) and by what shared memory feeds them, so what counts is how many products a thread makes of
// what it loads, how many places a load asks for, and that no product waits for the one in front. A block takes up to 64 query rows, (token, head-of-group) pairs
// of one key/value head of one request, and walks its keys 128 at a time. Its 256 threads are two halves, which share the keys, of 8 by 16: a thread has up to
// eight rows' scores with four keys (12 loads to 128 multiply-adds), then eight rows' sums of eight channels. Between them the scores lie in shared memory, where
// the softmax walks a row with four lanes. Where the blocks of rows are fewer than the device runs at once, a request's keys are shared by the blocks
// of a thread-block cluster, which join their sums, in the order of the keys, from one another's shared memory. Masked keys are skipped: nothing of them reaches a sum.
// Four trees of 12 over up to 1,024 keys of heads of 64: 26 us (128 threads, eight rows by eight keys each: 29; a half's lanes in two runs of sixteen instead of
// pairs: 27; copies of the next step's keys under this one's products: 27.5). 64 rows over 8,000 keys of 8 heads of 128: 120 (182, 134, 133.5).
// (Sixteen rows a warp, a lane a key: 47 for the former. Sums by products of pairs, fma.rn.f32x2: 28, and 127 for the latter.)
#include "branches.h"
#include "tc_common.cuh"

#include <type_traits>

namespace {

using branches::TreeParams;

constexpr int HALF = 128, THREADS = 2 * HALF;   // threads of a block: two halves, which share a row's keys
constexpr int ACROSS = 16;                      // threads of a row in each
constexpr int MOST_PARTS = 8;

// What a head size takes: rows of a block and keys of a step, rows and keys of a thread; in the second product how many threads share a row's keys, and the fours of
// channels of each (eight rows by eight channels, so that loads and multiply-adds take as long).
template <int HDMAX, int R>
struct Shape {
  static constexpr int ROWS = R * (HALF / ACROSS), KEYS = HDMAX > 128 ? 64 : 128, K = KEYS / (2 * ACROSS), WIDE = HDMAX > 64 ? ACROSS : ACROSS / 2;
  static constexpr int SPLIT = 2 * ACROSS / WIDE, FOURS = HDMAX / (4 * WIDE);
  static constexpr int SHARE = 32 / R, BATCH = KEYS / SHARE < 8 ? KEYS / SHARE : 8;       // lanes of a row in the softmax (a warp has R rows), and scores they have at a time
  static constexpr int P_LD = ROWS + 4;         // floats of a key's weights
};
// floats of a row of channels: an odd number of 16 bytes, so that eight lanes' rows lie on different banks
__host__ __device__ constexpr int row_floats(int hd) { return hd + (hd / 4 % 2 == 0 ? 4 : 8); }
// queries; keys, then weights; values
template <typename S>
__host__ __device__ constexpr int key_floats(int hd) {
  return S::KEYS * (row_floats(hd) > S::P_LD ? row_floats(hd) : S::P_LD);
}
template <typename S>
__host__ __device__ constexpr int smem_floats(int hd) {
  return S::ROWS * row_floats(hd) + key_floats<S>(hd) + S::KEYS * row_floats(hd);
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  gb::store_pair(p, v.x, v.y);
  gb::store_pair(p + 2, v.z, v.w);
}
// What stands for a masked key's score and weight: a NaN that no arithmetic gives (its results' are 0x7FFFFFFF), so that a key that is read counts whatever
// its score is: a weight of nothing times a value that is not finite is none.
constexpr uint32_t MASKED = 0xFFFFFFFFu;
__device__ __forceinline__ bool is_masked(float x) { return __float_as_uint(x) == MASKED; }
// exp of a difference; -inf gives 0
__device__ __forceinline__ float weight_of(float s, float m) { return m == -INFINITY ? 0.f : expf(s - m); }

__device__ __forceinline__ void copy_async_16(float* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

template <typename T, int HDMAX, int R>
__global__ void __launch_bounds__(THREADS, HDMAX <= 64 && R < 8 ? 2 : 1)
attention_tree_simple_kernel(const TreeParams p, const int hd, const int parts) {
  using S = Shape<HDMAX, R>;
  constexpr int ROWS = S::ROWS, KEYS = S::KEYS, K = S::K, FOURS = S::FOURS, WIDE = S::WIDE, P_LD = S::P_LD, BATCH = S::BATCH;
  extern __shared__ __align__(16) float smem[];
  __shared__ long long where[KEYS];            // the step's keys: their rows' places in the pools, -1: no page
  __shared__ float keep_s[ROWS];               // by what a row's sums are multiplied for a new maximum
  const int ld = row_floats(hd), c4 = hd / 4;
  float* const qs = smem;
  float* const ks = qs + ROWS * ld;            // keys, then the weights, a key's rows side by side
  float* const vs = ks + key_floats<S>(hd);
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  const int r = blockIdx.z, kvh = blockIdx.y % p.Hkv, block = blockIdx.y / p.Hkv, part = blockIdx.x;
  const int q_begin = p.cu_q[r], q_len = p.cu_q[r + 1] - q_begin, row0 = block * ROWS, nrows = min(ROWS, q_len * p.g - row0);
  const int kv_len = max(0, p.kv_lens[r]), ctx = max(0, kv_len - q_len);
  if (nrows <= 0) return;                      // (the whole cluster's)
  const int lo = (p.window > 0 ? max(0, ctx + 1 - p.window) : 0) / KEYS, steps = (kv_len - 1) / KEYS + 1 - lo;       // (one at least, without keys too)
  const int per = (steps + parts - 1) / parts, begin = lo + part * per, end = min(lo + steps, begin + per);
  const int32_t* table = p.block_table + (size_t)r * p.table_width;

  const int half = threadIdx.x / HALF, pair = threadIdx.x % HALF / 32;         // a warp of each half makes a pair: it has 2 R rows
  // Neighbouring lanes have two groups of rows, pairs of lanes the keys or channels: of a 16-byte load a quad of lanes asks for two places at most, for which
  // shared memory takes two clocks; with more it takes four.
  const int lane = threadIdx.x & 31, tx = lane / 2, first_row = (2 * pair + lane % 2) * R, channel0 = 4 * (tx % WIDE), split = half * (ACROSS / WIDE) + tx / WIDE;
  const int soft_row = (2 * pair + half) * R + lane % R, soft_share = lane / R;      // this lane's row in the softmax
  auto meet_pair = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + pair) : "memory"); };
  const bool there = soft_row < nrows;
  const int token = q_begin + (there ? (row0 + soft_row) / p.g : 0), start = p.window > 0 ? p.positions[token] + 1 - p.window : 0;
  const uint32_t* const bits = p.mask + (size_t)token * p.mask_words;
  // Rows to shared memory, eight threads a row at a time: 32-bit ones by asynchronous copies, others by way of registers
  auto fetch = [&](const void* pool, float* to) {
    for (int x = threadIdx.x / 8; x < KEYS; x += THREADS / 8) {
      const long long at = where[x];
      const T* const from = reinterpret_cast<const T*>(pool) + at;
#pragma unroll 2
      for (int c = threadIdx.x % 8; c < c4; c += 8) {
        float* const there = to + x * ld + c * 4;
        if (at < 0) *reinterpret_cast<float4*>(there) = make_float4(0.f, 0.f, 0.f, 0.f);
        else if (sizeof(T) == 4) copy_async_16(there, from + c * 4);
        else *reinterpret_cast<float4*>(there) = load4(from + c * 4);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const T* q = reinterpret_cast<const T*>(p.q);
  for (int x = threadIdx.x / 8; x < ROWS; x += THREADS / 8) {
    const int at = row0 + x;
    const T* const from = q + ((size_t)(q_begin + at / p.g) * p.Hq + kvh * p.g + at % p.g) * hd;
    for (int c = threadIdx.x % 8; c < c4; c += 8)
      *reinterpret_cast<float4*>(qs + x * ld + c * 4) = x < nrows ? load4(from + c * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int channel[FOURS];                          // this thread's fours of channels; those that the head does not have read another and are not stored
#pragma unroll
  for (int c = 0; c < FOURS; ++c) channel[c] = channel0 + 4 * WIDE * c < hd ? channel0 + 4 * WIDE * c : 0;
  float m = -INFINITY, l = 0.f;                // of this lane's row; the denominator: of its share of the keys
  float4 o[R][FOURS];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < FOURS; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);

  for (int step = begin; step < end; ++step) {
    const int key0 = step * KEYS;
    __syncthreads();                           // all are done with the step in front
    if (threadIdx.x < KEYS) {
      const int at = key0 + threadIdx.x, slot = at / p.page_size;
      const int page = at < kv_len && slot < p.table_width ? table[slot] : -1;
      where[threadIdx.x] = page >= 0 && page < p.pages ? (((long long)page * p.Hkv + kvh) * p.page_size + at % p.page_size) * hd : -1;
    }
    __syncthreads();
    fetch(p.k_pool, ks);
    fetch(p.v_pool, vs);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();                           // the keys are there
    // ---- scores of this thread's rows with keys tx, tx + 16, ...
    float s[R][K];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < K; ++e) s[i][e] = 0.f;
#pragma unroll 2
    for (int c = 0; c < c4; ++c) {
      float4 a[R], b[K];
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = *reinterpret_cast<const float4*>(qs + (first_row + i) * ld + c * 4);
#pragma unroll
      for (int e = 0; e < K; ++e) b[e] = *reinterpret_cast<const float4*>(ks + (tx + ACROSS * (half * K + e)) * ld + c * 4);
      // (channel by channel: a sum's next addition is 64 others later)
      auto add = [&](auto channel) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < K; ++e) s[i][e] = fmaf(channel(a[i]), channel(b[e]), s[i][e]);
      };
      add([](const float4& v) { return v.x; });
      add([](const float4& v) { return v.y; });
      add([](const float4& v) { return v.z; });
      add([](const float4& v) { return v.w; });
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                           // all have read the keys, and the values are there
#pragma unroll
    for (int e = 0; e < K; ++e)
#pragma unroll
      for (int i = 0; i < R; i += 2)
        *reinterpret_cast<float2*>(ks + (tx + ACROSS * (half * K + e)) * P_LD + first_row + i) = make_float2(s[i][e], s[i + 1][e]);
    meet_pair();                               // (a pair's rows are its own)
    // ---- the softmax, a row to one, two or four lanes, in loops: laid out over a thread's 64 scores it took six times as long, its instructions on their way
    const bool edge = key0 + KEYS > ctx || p.window > 0;
    float* const mine = ks + soft_row;
    float top = m;
#pragma unroll 1
    for (int k0 = soft_share; k0 < KEYS; k0 += BATCH * S::SHARE) {
      float x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) x[u] = mine[(k0 + u * S::SHARE) * P_LD] * p.scale;
      if (edge) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int k = k0 + u * S::SHARE, key = key0 + k, j = key - ctx;
          bool sees = there && key < kv_len;
          if (j < 0) sees = sees && key >= start;
          else sees = sees && (j >> 5) < p.mask_words && (bits[j >> 5] >> (j & 31) & 1u);
          if (!sees) x[u] = __uint_as_float(MASKED);
        }
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        mine[(k0 + u * S::SHARE) * P_LD] = x[u];
        top = fmaxf(top, x[u]);                // (of a number and a NaN the number)
      }
    }
#pragma unroll
    for (int d = R; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float keep = m == -INFINITY ? 1.f : weight_of(m, top), less = top == -INFINITY ? 0.f : top;        // (of nothing, or of what is no number and stays none)
    float sum = 0.f;
#pragma unroll 1
    for (int k0 = soft_share; k0 < KEYS; k0 += BATCH * S::SHARE) {
      float x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) x[u] = mine[(k0 + u * S::SHARE) * P_LD];
      // (a score that is no number stays none)
#pragma unroll
      for (int u = 0; u < BATCH; ++u) x[u] = is_masked(x[u]) ? x[u] : expf(x[u] - less);
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        sum += is_masked(x[u]) ? 0.f : x[u];
        mine[(k0 + u * S::SHARE) * P_LD] = x[u];
      }
    }
    l = l * keep + sum, m = top;
    if (soft_share == 0) keep_s[soft_row] = keep;
    meet_pair();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float less_now = keep_s[first_row + i];
      if (less_now != 1.f) {
#pragma unroll
        for (int c = 0; c < FOURS; ++c) o[i][c].x *= less_now, o[i][c].y *= less_now, o[i][c].z *= less_now, o[i][c].w *= less_now;
      }
    }
    // ---- sums of this thread's rows' channels, over its share of the keys, masked ones left out
    auto sums = [&](auto masked) {
      // (the next key's weights and values are on their way while this one's are multiplied: there may be no other warp to fill the wait)
      float w[2][R];
      float4 v[2][FOURS];
      auto load = [&](int key, float (&w)[R], float4 (&v)[FOURS]) {
        const float* const from = ks + key * P_LD + first_row;
        if constexpr (R % 4 == 0) {
#pragma unroll
          for (int i = 0; i < R; i += 4) {
            const float4 w4 = *reinterpret_cast<const float4*>(from + i);
            w[i] = w4.x, w[i + 1] = w4.y, w[i + 2] = w4.z, w[i + 3] = w4.w;
          }
        } else {
          const float2 w2 = *reinterpret_cast<const float2*>(from);
          w[0] = w2.x, w[1] = w2.y;
        }
#pragma unroll
        for (int c = 0; c < FOURS; ++c) v[c] = *reinterpret_cast<const float4*>(vs + key * ld + channel[c]);
      };
      auto add = [&](const float (&w)[R], const float4 (&v)[FOURS]) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (decltype(masked)::value && is_masked(w[i])) continue;
#pragma unroll
          for (int c = 0; c < FOURS; ++c) {
            o[i][c].x = fmaf(w[i], v[c].x, o[i][c].x), o[i][c].y = fmaf(w[i], v[c].y, o[i][c].y);
            o[i][c].z = fmaf(w[i], v[c].z, o[i][c].z), o[i][c].w = fmaf(w[i], v[c].w, o[i][c].w);
          }
        }
      };
      // an even number of keys a thread, those behind the last masked or (without masks) there; their rows are in shared memory in any case
      load(split, w[0], v[0]);
#pragma unroll 1
      for (int key = split; key < KEYS; key += 2 * S::SPLIT) {
        load(key + S::SPLIT, w[1], v[1]);
        add(w[0], v[0]);
        if (key + 2 * S::SPLIT < KEYS) load(key + 2 * S::SPLIT, w[0], v[0]);
        add(w[1], v[1]);
      }
    };
    if (edge) sums(std::true_type{});
    else sums(std::false_type{});
  }
#pragma unroll
  for (int d = R; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  // ---- every row's sums, maximum and denominator where the queries were; then the cluster's blocks join their shares of the rows
  __syncthreads();
  auto sums_to = [&](float* rows, bool add) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < FOURS; ++c) {
        float4* const to = reinterpret_cast<float4*>(rows + (first_row + i) * ld + channel0 + 4 * WIDE * c);
        const bool mine = tx < WIDE && channel0 + 4 * WIDE * c < hd;
        if (add && mine) {
          const float4 other = *reinterpret_cast<const float4*>(ks + (first_row + i) * ld + channel0 + 4 * WIDE * c);
          o[i][c].x += other.x, o[i][c].y += other.y, o[i][c].z += other.z, o[i][c].w += other.w;
        }
        if (mine) *to = o[i][c];
      }
  };
  if (WIDE < ACROSS) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < FOURS; ++c) {
        o[i][c].x += __shfl_xor_sync(0xffffffffu, o[i][c].x, 2 * WIDE), o[i][c].y += __shfl_xor_sync(0xffffffffu, o[i][c].y, 2 * WIDE);
        o[i][c].z += __shfl_xor_sync(0xffffffffu, o[i][c].z, 2 * WIDE), o[i][c].w += __shfl_xor_sync(0xffffffffu, o[i][c].w, 2 * WIDE);
      }
  }
  if (half == 1) sums_to(ks, false);                     // (where keys and weights were)
  __syncthreads();
  if (half == 0) sums_to(qs, true);
  if (soft_share == 0) *reinterpret_cast<float2*>(qs + soft_row * ld + hd) = make_float2(m, l);
  T* const out = reinterpret_cast<T*>(p.out);
  auto place = [&](int row) { return out + ((size_t)(q_begin + (row0 + row) / p.g) * p.Hq + kvh * p.g + (row0 + row) % p.g) * hd; };
  if (parts == 1) {
    __syncthreads();
    for (int x = threadIdx.x; x < nrows * c4; x += THREADS) {
      const int row = x / c4, c = x % c4;
      const float den = qs[row * ld + hd + 1], inv = den == 0.f ? 0.f : 1.0f / den;
      const float4 v = *reinterpret_cast<const float4*>(qs + row * ld + c * 4);
      store4(place(row) + c * 4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
    return;
  }
  tc::cluster_arrive_wait();
  for (int x = part * THREADS + threadIdx.x; x < nrows * c4; x += parts * THREADS) {
    const int row = x / c4, c = x % c4;
    const uint32_t v_at = tc::smem_u32(qs + row * ld + c * 4), ml_at = tc::smem_u32(qs + row * ld + hd);
    float2 ml[MOST_PARTS];
    float4 v[MOST_PARTS];
#pragma unroll
    for (int i = 0; i < MOST_PARTS; ++i) {
      const uint32_t from = min(i, parts - 1), a = tc::map_to_rank(ml_at, from), b = tc::map_to_rank(v_at, from);
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[i].x), "=f"(ml[i].y) : "r"(a) : "memory");
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[i].x), "=f"(v[i].y), "=f"(v[i].z), "=f"(v[i].w) : "r"(b) : "memory");
    }
    float mt = -INFINITY, lt = 0.f;
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < MOST_PARTS; ++i) {
      if (i >= parts || (ml[i].x == -INFINITY && ml[i].y == 0.f)) continue;        // no key of this part
      const float top = fmaxf(mt, ml[i].x), keep = mt == -INFINITY ? 1.f : weight_of(mt, top), add = ml[i].x == -INFINITY ? 1.f : weight_of(ml[i].x, top);
      t.x = t.x * keep + v[i].x * add, t.y = t.y * keep + v[i].y * add, t.z = t.z * keep + v[i].z * add, t.w = t.w * keep + v[i].w * add;
      lt = lt * keep + ml[i].y * add, mt = top;
    }
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    store4(place(row) + c * 4, make_float4(t.x * inv, t.y * inv, t.z * inv, t.w * inv));
  }
  tc::cluster_read_wait();                     // nobody leaves while another reads
}

// How a call is cut: the rows of a block (8 r), and the parts of a request's keys.
struct Plan {
  int r, parts;
  float time;
};

// Clusters of `parts` blocks that run at once.
template <typename T, int HDMAX, int R>
int at_once(int parts) {
  static branches::AskedOnce<MOST_PARTS + 1> known;
  return known.get(parts, [&] {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(parts), config.blockDim = dim3(THREADS), config.dynamicSmemBytes = 4 * smem_floats<Shape<HDMAX, R>>(HDMAX);
    cudaLaunchAttribute shape;
    shape.id = cudaLaunchAttributeClusterDimension;
    shape.val.clusterDim.x = parts, shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
    config.attrs = &shape, config.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, attention_tree_simple_kernel<T, HDMAX, R>, &config) != cudaSuccess) n = 0, cudaGetLastError();
    return n;
  });
}

template <typename T, int HDMAX, int R>
int configure() {
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(attention_tree_simple_kernel<T, HDMAX, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               4 * smem_floats<Shape<HDMAX, R>>(HDMAX));
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "tree_attention: %s", cudaGetErrorString(e));
    configured.done();
  }
  return GB_OK;
}

template <typename T, int HDMAX, int R>
int consider(const TreeParams& p, int max_q_len, int max_kv_len, float start, float step, Plan& best) {
  using S = Shape<HDMAX, R>;
  const int rc = configure<T, HDMAX, R>();
  const long long units = ((long long)max_q_len * p.g + S::ROWS - 1) / S::ROWS * p.Hkv * p.R;
  const int steps = (max_kv_len + S::KEYS - 1) / S::KEYS;
  for (int parts = 1; !rc && parts <= MOST_PARTS && (parts == 1 || parts <= steps); ++parts) {
    const int room = at_once<T, HDMAX, R>(parts);
    if (room == 0) continue;
    const float time = (float)((units + room - 1) / room) * (start + step * (float)((steps + parts - 1) / parts));
    if (time < best.time) best = Plan{R, parts, time};
  }
  return rc;
}

template <typename T, int HDMAX, int R>
int launch(const TreeParams& p, int hd, int max_q_len, int parts, cudaStream_t stream) {
  using S = Shape<HDMAX, R>;
  const long long blocks = ((long long)max_q_len * p.g + S::ROWS - 1) / S::ROWS;
  if (p.R > 65535 || blocks * p.Hkv > 65535) return gb::fail(GB_UNSUPPORTED, "tree_attention: %d requests, %lld blocks of rows", p.R, blocks * p.Hkv);
  return gb::check_pdl_launch(gb::launch_pdl(attention_tree_simple_kernel<T, HDMAX, R>, dim3(parts, (unsigned)(blocks * p.Hkv), p.R), dim3(THREADS),
                                             4 * smem_floats<S>(hd), stream, dim3(parts), p, hd, parts), "tree_attention");
}

// What takes least: all blocks in as many rounds as the device needs for them, each as long as a start and its steps. The figures are microseconds, measured with
// one block an SM (heads of 64 and, of 128 and 256 alike, 128 keys of 128 channels or 64 of 256). So 5 tokens without shared heads over 500 keys have blocks
// of 16 rows, two a request (20 us; 64 rows in one or two parts 80 and 43), 64 rows over 8,000 keys two blocks of 32 in six parts (120; 64 in
// eight parts, of which 15 run at once, 159).
template <typename T, int HDMAX>
int by_rows(const TreeParams& p, int hd, int max_q_len, int max_kv_len, cudaStream_t stream) {
  Plan best{0, 1, INFINITY};
  constexpr bool SMALL = HDMAX <= 64;
  int rc = consider<T, HDMAX, 2>(p, max_q_len, max_kv_len, SMALL ? 7.f : 8.f, SMALL ? 5.f : 9.f, best);
  if (!rc) rc = consider<T, HDMAX, 4>(p, max_q_len, max_kv_len, SMALL ? 7.f : 8.5f, SMALL ? 7.f : 12.f, best);
  if (!rc && HDMAX <= 128) rc = consider<T, HDMAX, (HDMAX > 128 ? 4 : 8)>(p, max_q_len, max_kv_len, SMALL ? 7.5f : 11.5f, SMALL ? 10.5f : 18.5f, best);
  if (rc) return rc;
  if (best.r == 2) return launch<T, HDMAX, 2>(p, hd, max_q_len, best.parts, stream);
  if (best.r == 8) return launch<T, HDMAX, (HDMAX > 128 ? 4 : 8)>(p, hd, max_q_len, best.parts, stream);
  return launch<T, HDMAX, 4>(p, hd, max_q_len, best.parts, stream);
}

}  // namespace

GB_EXPORT int gb_tree_attention_simple(const branches::TreeCall* call) {
  const TreeParams p = call->params();
  const int head_dim = (int)call->head_dim, max_q_len = (int)call->max_q_len, max_kv_len = (int)call->max_kv_len;
  if (head_dim % 4 != 0 || head_dim > 256) return gb::fail(GB_UNSUPPORTED, "tree_attention: heads of %d channels", head_dim);
  return GB_DISPATCH_DTYPE(call->dtype, E, [&]() -> int {
    if (head_dim <= 64) return by_rows<E, 64>(p, head_dim, max_q_len, max_kv_len, (cudaStream_t)call->stream);
    if (head_dim <= 128) return by_rows<E, 128>(p, head_dim, max_q_len, max_kv_len, (cudaStream_t)call->stream);
    return by_rows<E, 256>(p, head_dim, max_q_len, max_kv_len, (cudaStream_t)call->stream);
  });
}
