// What the attention kernels over pages of codes share: the argument block and who takes which request, the products of codes, a query as two
// rows of codes, the pools' tensor maps.
#pragma once

#include "float8.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace attn8 {

// A request with at most this many (token, head-of-group) rows is a decode request: each is two of a product's 16 (or 32) columns.
__host__ __device__ inline int decode_rows(int g) { return g <= 8 ? 8 : g <= 16 ? 16 : 0; }

struct Params {
  const __nv_bfloat16* q;        // [T, Hq, HD]
  const float *k_scale, *v_scale;        // [pages, Hkv]
  __nv_bfloat16* out;            // [T, Hq * HD]
  const int32_t* block_table;    // [R, table_width]
  const int32_t* cu_q;           // [R + 1]
  const int32_t* kv_lens;        // [R]
  int table_width, R, Hq, Hkv, g, window, page;
  float scale_log2;              // scale * log2(e)
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// Sums in 32 bits; E4M3 operands, or (the same bits, for the product of halves) halves.
__device__ __forceinline__ constexpr uint32_t instr_desc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Rows of 128 bytes (or of 64) as TMA swizzles them, eight to a group; for keys and queries the contraction lies along the row, for
// values the rows are the contraction.
template <int HD>
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t addr) {
  if (HD == 128) return tc::smem_desc_sw128(addr);
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(512 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
}
// Byte offset of 16-byte chunk `c` of row `row` in such a tile.
template <int HD>
__device__ __forceinline__ uint32_t swizzled(int row, int c) {
  return HD == 128 ? (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}

// A lane's part of a query row, two bfloat16 numbers a word, LANES neighbouring lanes a row, as codes: the row over 2^e, by a power of two at a largest
// of at most 448, and `finer` times what these leave. 2^e.
template <int LANES, int WORDS>
__device__ __forceinline__ float split_query(const uint32_t (&w)[WORDS], float finer, uint32_t (&hi)[WORDS / 2], uint32_t (&lo)[WORDS / 2]) {
  float v[2 * WORDS], largest = 0.f;
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    largest = max3(largest, fabsf(v[2 * i]), fabsf(v[2 * i + 1]));
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  const int e = f8::scale_exponent(largest);
  // (scores with an infinite channel are infinite or no numbers, and their softmax is no number)
  const float inv = largest < INFINITY ? f8::power_of_two(-e) : NAN;
#pragma unroll
  for (int i = 0; i < WORDS / 2; ++i) {
    const float a = v[4 * i] * inv, b = v[4 * i + 1] * inv, c = v[4 * i + 2] * inv, d = v[4 * i + 3] * inv;
    hi[i] = f8::encode4(a, b, c, d);
    const float4 back = f8::decode4(hi[i]);
    lo[i] = f8::encode4(finer * (a - back.x), finer * (b - back.y), finer * (c - back.z), finer * (d - back.w));
  }
  return f8::power_of_two(e);
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
inline int pool_map(const void* ptr, int page, int heads, long long pages, int hd, CUtensorMap* out) {
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

}  // namespace attn8
