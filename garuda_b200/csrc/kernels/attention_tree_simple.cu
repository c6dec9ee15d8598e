// Attention of drafted trees over the paged cache in 32-bit arithmetic throughout: the true 32-bit path, and bfloat16 where the kernel on
// the tensor cores does not apply (head sizes other than 64 and 128, pages of other sizes). The same formula, see attention_tree_tcgen05.cu.
//
// Bound by the multiply-adds (32-bit ones run on the ordinary pipes): a block takes 32 query rows, (token, head-of-group) pairs of
// one key/value head of one request, and walks its keys 32 at a time, so that a number from shared memory is used eight times in each
// product. Its 128 threads are 16 pairs of rows by 8: a thread has two rows' scores with four keys, and of the sums two rows' every eighth four
// channels. A row's eight threads are neighbours of one warp: maxima and sums are three shuffles, and the weights need no barrier.
// Where the blocks of rows are fewer than the device runs at once, a request's keys are shared by the blocks of a thread-block cluster, which join their
// sums, in the order of the keys, from one another's shared memory. Masked keys are skipped: nothing of them reaches a sum.
#include "branches.h"
#include "tc_common.cuh"

namespace {

using branches::TreeParams;

constexpr int ROWS = 32, KEYS = 32, THREADS = 128;
constexpr int P_LD = KEYS + 4;
constexpr int MOST_PARTS = 8;

__host__ __device__ constexpr int row_floats(int hd) { return hd + 4; }        // (eight rows' 16 bytes on different banks where hd is a multiple of 32)
__host__ __device__ constexpr int smem_floats(int hd) { return (ROWS + 4 * KEYS) * row_floats(hd) + ROWS * P_LD; }

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
// exp of a difference; -inf gives 0
__device__ __forceinline__ float weight_of(float s, float m) { return m == -INFINITY ? 0.f : expf(s - m); }

__device__ __forceinline__ void copy_async_16(float* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

template <typename T, int HDMAX>
__global__ void __launch_bounds__(THREADS)
attention_tree_simple_kernel(const TreeParams p, const int hd, const int parts) {
  constexpr int MOST = HDMAX / 32;             // fours of channels that a thread sums
  extern __shared__ __align__(16) float smem[];
  __shared__ long long where[2][KEYS];         // two tiles' keys: their rows' places in the pools, -1: no page
  const int ld = row_floats(hd), c4 = hd / 4;
  float* const qs = smem;
  float* const ring = qs + ROWS * ld;          // two tiles: keys, then values
  float* const ps = ring + 4 * KEYS * ld;
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  const int r = blockIdx.z, kvh = blockIdx.y % p.Hkv, block = blockIdx.y / p.Hkv, part = blockIdx.x;
  const int q_begin = p.cu_q[r], q_len = p.cu_q[r + 1] - q_begin, row0 = block * ROWS, nrows = min(ROWS, q_len * p.g - row0);
  const int kv_len = p.kv_lens[r], ctx = max(0, kv_len - q_len);
  if (nrows <= 0 || kv_len <= 0) return;       // (the whole cluster's)
  const int lo = (p.window > 0 ? max(0, ctx + 1 - p.window) : 0) / KEYS, tiles = (kv_len - 1) / KEYS + 1 - lo;
  const int per = (tiles + parts - 1) / parts, tile_begin = lo + part * per, tile_end = min(lo + tiles, tile_begin + per);
  const int32_t* table = p.block_table + (size_t)r * p.table_width;

  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  auto place_keys = [&](int tile) {            // by the first warp
    if (threadIdx.x < KEYS && tile < tile_end) {
      const int at = tile * KEYS + threadIdx.x, slot = at / p.page_size;
      const int page = at < kv_len && slot < p.table_width ? table[slot] : -1;
      where[tile & 1][threadIdx.x] =
          page >= 0 && page < p.pages ? (((long long)page * p.Hkv + kvh) * p.page_size + at % p.page_size) * hd : -1;
    }
  };
  // A tile's keys and values: 32-bit ones on their way to shared memory while the tile in front is at work, others by way of registers
  auto fetch = [&](int tile) {
    float* const ks = ring + (tile & 1) * 2 * KEYS * ld;
#pragma unroll 4
    for (int x = threadIdx.x; x < 2 * KEYS * c4; x += THREADS) {
      const int half = x >= KEYS * c4, y = x - half * KEYS * c4, key = y / c4, c = y % c4;
      const long long at = where[tile & 1][key];
      float* const to = ks + (half * KEYS + key) * ld + c * 4;
      const T* const from = reinterpret_cast<const T*>(half ? p.v_pool : p.k_pool) + at + c * 4;
      if (at < 0) *reinterpret_cast<float4*>(to) = make_float4(0.f, 0.f, 0.f, 0.f);
      else if (sizeof(T) == 4) copy_async_16(to, from);
      else *reinterpret_cast<float4*>(to) = load4(from);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const T* q = reinterpret_cast<const T*>(p.q);
  place_keys(tile_begin);
  place_keys(tile_begin + 1);
  __syncthreads();
  if (tile_begin < tile_end) fetch(tile_begin);
  for (int x = threadIdx.x; x < ROWS * c4; x += THREADS) {
    const int row = x / c4, c = x % c4, at = row0 + row;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < nrows) v = load4(q + ((size_t)(q_begin + at / p.g) * p.Hq + kvh * p.g + at % p.g) * hd + c * 4);
    *reinterpret_cast<float4*>(qs + row * ld + c * 4) = v;
  }
  // this thread's two rows
  int token[2], start[2];
  bool there[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = 2 * ty + i;
    there[i] = row < nrows;
    token[i] = q_begin + (there[i] ? (row0 + row) / p.g : 0);
    start[i] = p.window > 0 ? p.positions[token[i]] + 1 - p.window : 0;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float4 o[2][MOST];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < MOST; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);

  for (int tile = tile_begin; tile < tile_end; ++tile) {
    const int key0 = tile * KEYS;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                           // the tile is there, and all are done with the one in front
    if (tile + 1 < tile_end) fetch(tile + 1);
    place_keys(tile + 2);
    const float* const ks = ring + (tile & 1) * 2 * KEYS * ld;
    const float* const vs = ks + KEYS * ld;
    // ---- scores of two rows with keys tx, tx + 8, tx + 16, tx + 24
    float s[2][4] = {};
#pragma unroll 4
    for (int c = 0; c < c4; ++c) {
      float4 a[2], b[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) a[i] = *reinterpret_cast<const float4*>(qs + (2 * ty + i) * ld + c * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = *reinterpret_cast<const float4*>(ks + (tx + 8 * e) * ld + c * 4);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = fmaf(a[i].x, b[e].x, s[i][e]);
          s[i][e] = fmaf(a[i].y, b[e].y, s[i][e]);
          s[i][e] = fmaf(a[i].z, b[e].z, s[i][e]);
          s[i][e] = fmaf(a[i].w, b[e].w, s[i][e]);
        }
    }
    // ---- the keys that a row does not read, then the softmax's running maximum and sum
    const bool edge = key0 + KEYS > ctx || p.window > 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float top = m[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] *= p.scale;
        if (edge) {
          const int key = key0 + tx + 8 * e, j = key - ctx;
          bool sees = there[i] && key < kv_len;
          if (j < 0) sees = sees && key >= start[i];
          else sees = sees && (j >> 5) < p.mask_words && (p.mask[(size_t)token[i] * p.mask_words + (j >> 5)] >> (j & 31) & 1u);
          if (!sees) s[i][e] = -INFINITY;
        }
        top = fmaxf(top, s[i][e]);
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float keep = weight_of(m[i], top);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (a masked key's weight is nothing, whatever the maximum is; a score that is no number stays none)
        const float w = s[i][e] == -INFINITY ? 0.f : expf(s[i][e] - (top == -INFINITY ? 0.f : top));
        sum += w;
        ps[(2 * ty + i) * P_LD + tx + 8 * e] = w;
      }
      l[i] = l[i] * (m[i] == -INFINITY ? 1.f : keep) + sum;          // this thread's share
      if (m[i] != -INFINITY && keep != 1.f) {
#pragma unroll
        for (int c = 0; c < MOST; ++c) o[i][c].x *= keep, o[i][c].y *= keep, o[i][c].z *= keep, o[i][c].w *= keep;
      }
      m[i] = top;
    }
    __syncwarp();
    // ---- sums of two rows' channels 4 tx + 32 c
#pragma unroll 2
    for (int key = 0; key < KEYS; key += 4) {
      const float4 w0 = *reinterpret_cast<const float4*>(ps + 2 * ty * P_LD + key), w1 = *reinterpret_cast<const float4*>(ps + (2 * ty + 1) * P_LD + key);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u0 = e == 0 ? w0.x : e == 1 ? w0.y : e == 2 ? w0.z : w0.w, u1 = e == 0 ? w1.x : e == 1 ? w1.y : e == 2 ? w1.z : w1.w;
#pragma unroll
        for (int c = 0; c < MOST; ++c) {
          if (4 * tx + 32 * c >= hd) break;
          const float4 v = *reinterpret_cast<const float4*>(vs + (key + e) * ld + 4 * tx + 32 * c);
          if (!edge || u0 != 0.f)
            o[0][c].x = fmaf(u0, v.x, o[0][c].x), o[0][c].y = fmaf(u0, v.y, o[0][c].y), o[0][c].z = fmaf(u0, v.z, o[0][c].z), o[0][c].w = fmaf(u0, v.w, o[0][c].w);
          if (!edge || u1 != 0.f)
            o[1][c].x = fmaf(u1, v.x, o[1][c].x), o[1][c].y = fmaf(u1, v.y, o[1][c].y), o[1][c].z = fmaf(u1, v.z, o[1][c].z), o[1][c].w = fmaf(u1, v.w, o[1][c].w);
        }
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
  T* const out = reinterpret_cast<T*>(p.out);
  auto place = [&](int row) { return out + ((size_t)(q_begin + (row0 + row) / p.g) * p.Hq + kvh * p.g + (row0 + row) % p.g) * hd; };
  if (parts == 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];
#pragma unroll
      for (int c = 0; c < MOST; ++c)
        if (there[i] && 4 * tx + 32 * c < hd)
          store4(place(2 * ty + i) + 4 * tx + 32 * c, make_float4(o[i][c].x * inv, o[i][c].y * inv, o[i][c].z * inv, o[i][c].w * inv));
    }
    return;
  }
  // ---- the cluster's parts: every row's sums, maximum and denominator where the tiles were, then each block joins its share of the rows
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float* to = ring + (2 * ty + i) * ld;
#pragma unroll
    for (int c = 0; c < MOST; ++c)
      if (4 * tx + 32 * c < hd) *reinterpret_cast<float4*>(to + 4 * tx + 32 * c) = o[i][c];
    if (tx == 0) to[hd] = m[i], to[hd + 1] = l[i];
  }
  tc::cluster_arrive_wait();
  for (int x = part * THREADS + threadIdx.x; x < nrows * c4; x += parts * THREADS) {
    const int row = x / c4, c = x % c4;
    const uint32_t v_at = tc::smem_u32(ring + row * ld + c * 4), ml_at = tc::smem_u32(ring + row * ld + hd);
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
  tc::cluster_arrive_wait();                   // nobody leaves while another reads
}

// Parts of a request's keys, a power of two: as many as fill the device four times over, each of two tiles at least.
int parts_of(long long units, int max_kv_len) {
  const int tiles = (max_kv_len + KEYS - 1) / KEYS;
  int parts = 1;
  while (parts < MOST_PARTS && 2 * parts * units <= 4ll * gb::sm_count() && 4 * parts <= tiles) parts *= 2;
  return parts;
}

template <typename T, int HDMAX>
int launch(const TreeParams& p, int hd, int blocks, int parts, cudaStream_t stream) {
  static gb::OncePerDevice configured;
  if (configured.needed()) {
    const cudaError_t e = cudaFuncSetAttribute(attention_tree_simple_kernel<T, HDMAX>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               4 * smem_floats(HDMAX));
    if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "tree_attention: %s", cudaGetErrorString(e));
    configured.done();
  }
  return gb::check_pdl_launch(gb::launch_pdl(attention_tree_simple_kernel<T, HDMAX>, dim3(parts, blocks * p.Hkv, p.R), dim3(THREADS),
                                             4 * smem_floats(hd), stream, dim3(parts), p, hd, parts), "tree_attention");
}

}  // namespace

GB_EXPORT int gb_tree_attention_simple(const branches::TreeCall* call) {
  const TreeParams p = call->params();
  const int R = p.R, Hkv = p.Hkv, head_dim = (int)call->head_dim;
  const long long blocks = (call->max_q_len * p.g + ROWS - 1) / ROWS;
  if (head_dim % 4 != 0 || head_dim > 256) return gb::fail(GB_UNSUPPORTED, "tree_attention: heads of %d channels", head_dim);
  if (R > 65535 || blocks * Hkv > 65535) return gb::fail(GB_UNSUPPORTED, "tree_attention: %d requests, %lld blocks of rows", R, blocks * Hkv);
  const int parts = parts_of(R * blocks * Hkv, (int)call->max_kv_len);
  return GB_DISPATCH_DTYPE(call->dtype, E, [&]() -> int {
    if (head_dim <= 64) return launch<E, 64>(p, head_dim, (int)blocks, parts, (cudaStream_t)call->stream);
    if (head_dim <= 128) return launch<E, 128>(p, head_dim, (int)blocks, parts, (cudaStream_t)call->stream);
    return launch<E, 256>(p, head_dim, (int)blocks, parts, (cudaStream_t)call->stream);
  });
}
