// Selection over beams and vocabulary: of an item's candidates (beam w, token v) with the scores
//   s_w + (x_wv - log sum_u exp x_wu)
// the K best, equal ones in the order of w * V + v. A beam whose score is not finite is over, one whose logits hold an infinity or
// NaN (or nothing but -inf) has no distribution: all their candidates count as -inf, as a token of logit -inf does.
//
// Bound by the one pass over the logits. Within a beam candidates lie as their logits do, so a block takes a stretch of a row into registers,
// finds its K largest logits and what the stretch adds to the row's sum, and leaves both in scratch memory; the block that counts the last
// of an item's stretches joins them. Rows of beams that are over are not read.
//   * The K largest: the maxima of at least K groups of threads are at hand, the K-th largest of these is no larger than the K-th largest logit, so
//     whatever is no smaller goes to a short list (2 to 4 K entries as a rule), where each entry counts those in front of it. A list that runs over
//     (many equal logits) is made again with the K-th key itself, found bit by bit.
//   * Two candidates of different beams may be as near as 1e-7, so sums and scores are in 64 bits where it matters: exponentials of the list's
//     entries, which are the large ones, and the sums over threads; a thread's other exponentials and its sum of 8 to 32 of them are 32-bit, whose errors
//     are of single terms that are each smaller than K others, and average out.
#include <climits>

#include "common.cuh"

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MOST = 64;             // candidates that are chosen, and beams
constexpr int LIST = 1024;           // entries of a short list

typedef unsigned long long Key;      // the larger logit first, then the smaller number: a block's keys all differ

__device__ __forceinline__ uint32_t ordered(float x) {               // unsigned numbers in the order of the floats (no NaN)
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }
__device__ __forceinline__ Key key_of(float x, int index) { return (Key)ordered(x + 0.f) << 32 | (0xFFFFFFFFu - (uint32_t)index); }   // (-0 is 0)
__device__ __forceinline__ float logit_of(Key k) { return from_ordered((uint32_t)(k >> 32)); }
__device__ __forceinline__ int index_of(Key k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Part {
  double top, sum;        // a stretch's largest logit, and the sum of exp(x - top)
};

struct Scored {
  double score;
  long long at;           // w * V + v
};
__device__ __forceinline__ bool in_front(double a, long long at, double b, long long bt) { return a > b || (a == b && at < bt); }

struct Shared {
  union {
    Key list[LIST];
    struct {
      double score[LIST];
      long long at[LIST];
      double head[THREADS];
    } join;
  };
  float group[MOST];
  double warp[WARPS], lse[MOST];
  float score[MOST];
  Scored won[MOST], reduce[WARPS];
  float top, least;
  double join_least;
  int n, last, taken[MOST];
};

// VALUES: logits a thread holds.
template <int VALUES>
__global__ void __launch_bounds__(THREADS)
beam_select_kernel(const float* __restrict__ logits, const long long ld, const float* __restrict__ scores, const int V, const int beams, const int K,
                   float* __restrict__ best, int32_t* __restrict__ parents, int32_t* __restrict__ tokens, Part* __restrict__ parts,
                   Key* __restrict__ lists, int* __restrict__ counters) {
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunk = blockIdx.x, chunks = gridDim.x, item = blockIdx.y / beams;
  const long long row = blockIdx.y;
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  if (is_finite(scores[row])) {
    // ---- a stretch of the row, in 16-byte loads: places count from the 16 bytes in which the row begins
    const float* const x_row = logits + row * ld;
    const int shift = (int)((uintptr_t)x_row >> 2 & 3);
    float x[VALUES];
    const int place0 = chunk * THREADS * VALUES + threadIdx.x * 4 - shift;       // of the first vector; the others THREADS * 4 apart
#pragma unroll
    for (int j = 0; j < VALUES / 4; ++j) {
      const int at = place0 + j * THREADS * 4;
      if (at >= 0 && at + 3 < V) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(x_row + at));
        x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * j + e] = at + e >= 0 && at + e < V ? x_row[at + e] : -INFINITY;
      }
    }
    auto place = [&](int i) { return place0 + (i >> 2) * THREADS * 4 + (i & 3); };
    // ---- a bound below the K-th largest: maxima of 16 warps, 32 halves or 64 quarters of one
    float top = x[0];
#pragma unroll
    for (int i = 1; i < VALUES; ++i) top = fmaxf(top, x[i]);
    const int groups = K <= 16 ? 16 : K <= 32 ? 32 : 64, width = THREADS / groups;
    for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (threadIdx.x % width == 0) sh.group[threadIdx.x / width] = top;
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    if (threadIdx.x < groups) {
      const float mine = sh.group[threadIdx.x];
      int rank = 0;
      for (int g = 0; g < groups; ++g) rank += sh.group[g] > mine || (sh.group[g] == mine && g < (int)threadIdx.x);
      if (rank == K - 1) sh.least = mine;
      if (rank == 0) sh.top = mine;
    }
    __syncthreads();
    const float block_top = sh.top, reference = -block_top * 1.4426950408889634f;
    float least = sh.least;
    Key exactly = 0;                       // 0: by the bound
    double sum;
    for (;;) {
      float rest[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        const bool listed = exactly ? x[i] > -INFINITY && key_of(x[i], place(i)) >= exactly : x[i] >= least && x[i] > -INFINITY;
        if (listed) {
          const int at = atomicAdd(&sh.n, 1);
          if (at < LIST) sh.list[at] = key_of(x[i], place(i));
        } else if (!(x[i] == -INFINITY)) {
          rest[i & 3] += fast_exp2(fmaf(x[i], 1.4426950408889634f, reference));
        }
      }
      sum = (double)((rest[0] + rest[1]) + (rest[2] + rest[3]));
      __syncthreads();
      if (sh.n <= LIST) break;
      // the K-th key, from its highest bit down: the largest number that K keys are no smaller than
      Key found = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const Key trial = found | (Key)1 << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) n += x[i] > -INFINITY && key_of(x[i], place(i)) >= trial;
        n = __reduce_add_sync(0xffffffffu, n);
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        if (lane == 0) atomicAdd(&sh.n, n);
        __syncthreads();
        if (sh.n >= K) found = trial;
      }
      __syncthreads();
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      exactly = found;
    }
    // ---- the list's entries: exponentials in 64 bits, and their places
    const int n = sh.n;
    Key* const list = lists + (row * chunks + chunk) * K;
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const Key mine = sh.list[i];
      sum += exp((double)logit_of(mine) - (double)block_top);
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sh.list[j] > mine;
      if (rank < K) list[rank] = mine;
    }
    for (int i = n + threadIdx.x; i < K; i += THREADS) list[i] = 0;
    sum = warp_sum(sum);
    if (lane == 0) sh.warp[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.;
      for (int w = 0; w < WARPS; ++w) all += sh.warp[w];
      parts[row * chunks + chunk] = Part{(double)block_top, all};
    }
  }
  // ---- the item's last block joins the stretches
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int seen = atomicAdd(&counters[item], 1);
    sh.last = seen == beams * chunks - 1;
    if (sh.last) counters[item] = 0;              // as the next launch expects it
  }
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  const long long row0 = (long long)item * beams;
  for (int w = warp; w < beams; w += WARPS) {
    const float score = scores[row0 + w];
    double lse = NAN;
    if (is_finite(score)) {
      double top = -INFINITY;
      for (int c = lane; c < chunks; c += 32) top = fmax(top, __ldcg(&parts[(row0 + w) * chunks + c].top));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      double all = 0.;
      for (int c = lane; c < chunks; c += 32) {
        const Part* part = &parts[(row0 + w) * chunks + c];
        const double t = __ldcg(&part->top), s = __ldcg(&part->sum);
        all += t == -INFINITY ? s : s * exp(t - top);            // (without a finite logit s is 0 or no number)
      }
      all = warp_sum(all);
      lse = log(all) + top;
    }
    if (lane == 0) sh.score[w] = score, sh.lse[w] = isfinite(lse) ? lse : NAN;
  }
  if (threadIdx.x == 0) sh.n = 0, sh.join_least = -INFINITY;
  __syncthreads();
  // ---- a bound below the K-th best: the lists are in order, so it is no worse than the K-th best of their heads (a thread's lists count as one)
  const int n_lists = beams * chunks, heads = min(n_lists, THREADS);
  auto entry = [&](int l, int i, double& score, long long& at) {           // the i-th of list l; false: it has no more
    const int w = l / chunks;
    if (i >= K || isnan(sh.lse[w])) return false;
    const Key k = __ldcg(&lists[(row0 * chunks + l) * K + i]);
    if (k == 0) return false;
    score = (double)sh.score[w] + ((double)logit_of(k) - sh.lse[w]);
    at = (long long)w * V + index_of(k);
    return true;
  };
  if ((int)threadIdx.x < heads) {
    double mine = -INFINITY, score;
    long long at;
    for (int l = threadIdx.x; l < n_lists; l += THREADS)
      if (entry(l, 0, score, at)) mine = fmax(mine, score);
    sh.join.head[threadIdx.x] = mine;
  }
  __syncthreads();
  if ((int)threadIdx.x < heads) {
    const double mine = sh.join.head[threadIdx.x];
    int rank = 0;
    for (int j = 0; j < heads; ++j) rank += sh.join.head[j] > mine || (sh.join.head[j] == mine && j < (int)threadIdx.x);
    if (rank == K - 1) sh.join_least = mine;
  }
  __syncthreads();
  const double least = sh.join_least;
  for (int l = threadIdx.x; l < n_lists; l += THREADS) {
    double score;
    long long at;
    for (int i = 0; entry(l, i, score, at) && score >= least; ++i) {
      const int slot = atomicAdd(&sh.n, 1);
      if (slot < LIST) sh.join.score[slot] = score, sh.join.at[slot] = at;
    }
  }
  __syncthreads();
  int found = min(sh.n, K);
  if (sh.n <= LIST) {
    const int n = sh.n;
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const double mine = sh.join.score[i];
      const long long at = sh.join.at[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += in_front(sh.join.score[j], sh.join.at[j], mine, at);
      if (rank < K) sh.won[rank] = Scored{mine, at};
    }
    __syncthreads();
  } else {
    // more than the short list holds (many equal scores): one after the other, each the best of those behind the one in front of it
    Scored last{INFINITY, -1};
    for (int r = 0; r < K; ++r) {
      Scored mine{-INFINITY, LLONG_MAX};
      for (int l = threadIdx.x; l < n_lists; l += THREADS) {
        double score;
        long long at;
        for (int i = 0; entry(l, i, score, at); ++i)
          if (in_front(last.score, last.at, score, at)) {
            if (in_front(score, at, mine.score, mine.at)) mine = Scored{score, at};
            break;
          }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double s = __shfl_xor_sync(0xffffffffu, mine.score, o);
        const long long a = __shfl_xor_sync(0xffffffffu, mine.at, o);
        if (in_front(s, a, mine.score, mine.at)) mine = Scored{s, a};
      }
      if (lane == 0) sh.reduce[warp] = mine;
      __syncthreads();
      mine = sh.reduce[0];
      for (int w = 1; w < WARPS; ++w)
        if (in_front(sh.reduce[w].score, sh.reduce[w].at, mine.score, mine.at)) mine = sh.reduce[w];
      if (threadIdx.x == 0) sh.won[r] = mine;
      last = mine;
      __syncthreads();
    }
  }
  // ---- fewer candidates than are asked for: of those of score -inf the first ones (of K numbers at least as many are not chosen yet)
  if (found < K) {
    for (int f = threadIdx.x; f < K; f += THREADS) {
      bool taken = false;
      for (int i = 0; i < found; ++i) taken = taken || sh.won[i].at == f;
      sh.taken[f] = taken;
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int f = 0, i = found; i < K; ++f)
        if (!sh.taken[f]) sh.won[i++] = Scored{-INFINITY, f};
    __syncthreads();
  }
  for (int i = threadIdx.x; i < K; i += THREADS) {
    const Scored s = sh.won[i];
    const long long out = (long long)item * K + i;
    best[out] = (float)s.score, parents[out] = (int)(s.at / V), tokens[out] = (int)(s.at % V);
  }
}

// How a row is cut: logits a thread holds. As many as leave the device two blocks an SM, so that the lists to join are few; as few as that
// takes, so that a small call is spread out.
int values_of(int rows, int V) {
  const int want = 2 * gb::sm_count();
  for (int values = 32; values > 4; values /= 2)
    if ((long long)rows * ((V + 3 + THREADS * values - 1) / (THREADS * values)) >= want) return values;
  return 4;
}
int chunks_of(int values, int V) { return (V + 3 + THREADS * values - 1) / (THREADS * values); }

}  // namespace

// Bytes of scratch memory of a call, of which the first `counter_bytes` (a counter for every item) are zero before the first one; every call
// leaves them zero.
GB_EXPORT long long gb_beam_select_scratch_bytes(int items, int beams, int V, int K, long long* counter_bytes) {
  const long long rows = (long long)items * beams, chunks = chunks_of(values_of((int)rows, V), V);
  *counter_bytes = ((long long)items * 4 + 15) / 16 * 16;
  return rows * chunks * (long long)(sizeof(Part) + K * sizeof(Key));
}

GB_EXPORT int gb_beam_select(const float* logits, long long ld, const float* scores, int items, int beams, int V, int K, float* best, int32_t* parents,
                             int32_t* tokens, void* counters, void* scratch, void* stream) {
  if (K > MOST || beams > MOST) return gb::fail(GB_UNSUPPORTED, "beam_select: %d of %d beams (at most %d)", K, beams, MOST);
  const int rows = items * beams, values = values_of(rows, V), chunks = chunks_of(values, V);
  if (rows > 65535) return gb::fail(GB_UNSUPPORTED, "beam_select: %d rows of logits", rows);
  Part* parts = reinterpret_cast<Part*>(scratch);
  Key* lists = reinterpret_cast<Key*>(parts + (long long)rows * chunks);
  const auto kernel = values == 32 ? beam_select_kernel<32> : values == 16 ? beam_select_kernel<16> : values == 8 ? beam_select_kernel<8> : beam_select_kernel<4>;
  return gb::check_pdl_launch(gb::launch_pdl(kernel, dim3(chunks, rows), dim3(THREADS), 0, (cudaStream_t)stream, dim3(1), logits, ld, scores, V,
                                             beams, K, best, parents, tokens, parts, lists, reinterpret_cast<int*>(counters)), "beam_select");
}
