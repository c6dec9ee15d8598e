// Selection over beams and vocabulary: of an item's candidates (beam w, token v) with the scores
//   s_w + (x_wv - log sum_u exp x_wu)
// the K best, equal ones in the order of w * V + v (beams of the same logits and score have the same ones, to the last bit). A beam whose score
// is not finite is over, one whose logits hold an infinity or NaN (or nothing but -inf) has no distribution: all their candidates count as -inf,
// as a token of logit -inf does.
//
// Bound by the one pass over the logits. Within a beam candidates lie as their logits do, so a block walks a stretch of a row, 4,096 (few: 1,024)
// logits at a time, and leaves its K largest and what the stretch adds to the row's sum in scratch memory; the block that counts the last
// of an item's stretches joins them. Of rows of beams that are over only the first tiles are read. Tiles come by bulk copies, one ahead (registers for that were
// spilled: 150 us against 56 for 512 rows of 128,256, whose bytes take 40); a thread's sixteen logits cost one comparison as long as none is above the
// bound. SMs with three rows are through with the stream some fifteen before those with four, and joining the last item takes five. A small
// call is a chain of waits: 4 rows of 32,000 take 8 us, half a one for the first tile, one for its bound, one for the list in order, one for the count, three
// and a half to join.
//   * The K largest: a list in shared memory of the logits above a bound. The first bound is the K-th largest of 64 maxima of groups of four
//     threads, which is no larger than the K-th largest logit; the list is cut to K, and its last entry becomes the bound, whenever it has grown. A tile
//     that runs the list over (many equal logits) enters by its own K-th key, found bit by bit.
//   * Two candidates of different beams may be as near as 1e-7, so sums and scores are in 64 bits where it matters: exponentials of what is on the
//     list at last, the largest ones, and the sum over tiles and threads; a thread's other exponentials of a tile and their sum are 32-bit:
//     a term that lies d below the largest logit is off by up to 2^-22 + 1.35e-7 d of itself (the exponential's error; the difference's and its product's roundings, log2(e)'s).
//     Errors of different terms average out (4e-8 at most in 600 draws of rows in four orders; with references up to 30 below the largest logit 4e-7 on ascending
//     rows). Those of equal ones do not: a row of one large logit and others d below is off by as much, and two roundings of a thread's sum, times their share of
//     the sum: below 2^-21 + 1.35e-7 d (5e-7 seen at d = 11 for 128,256 of them).
#include <climits>
#include <type_traits>

#include "error_word.cuh"
#include "tc_common.cuh"

namespace {

using namespace tc;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MANY = 16;             // logits a thread holds of a tile (of a small call 4)
constexpr int STAGES = 2;            // tiles in shared memory
constexpr int GROUPS = 64;           // of threads, for the first bound
constexpr int BLOCKS_PER_SM = 4;
constexpr int MOST = 64;             // candidates that are chosen, and beams
constexpr int LIST = 512;            // entries of a list
constexpr int JOINED = 1024 + 64;    // of the list of all beams' candidates
constexpr float CLOSE = 1.f;         // a reference may stay this far below the largest logit (its distance is what a term's exponent is rounded by)

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
__device__ __noinline__ double exp_of(double x) { return exp(x); }         // (many instructions: once)
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Joined {           // where the ring was
  double score[JOINED];
  long long at[JOINED];
};

struct Part {
  double ref, sum;        // a stretch's sum of exp(x - ref); its largest logit is at most CLOSE above ref
};

struct Scored {
  double score;
  long long at;           // w * V + v
};
__device__ __forceinline__ bool in_front(double a, long long at, double b, long long bt) { return a > b || (a == b && at < bt); }

__device__ __forceinline__ float2 add2(float2 a, float2 b) {          // two at a time
  float2 d;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

struct Shared {
  uint64_t full[STAGES];
  Key list[2][LIST];
  float group[GROUPS];
  double warp[WARPS], lse[MOST];
  float score[MOST];
  Scored won[MOST];
  float top, bound;
  int n, last, taken[MOST];
};

// The four neighbouring threads of an entry count together: how many of them say so, to all four.
__device__ __forceinline__ int sum_of_four(int n) {
  n += __shfl_xor_sync(0xffffffffu, n, 1);
  return n + __shfl_xor_sync(0xffffffffu, n, 2);
}
// The maxima of the 64 groups of four threads into sh.group; the K-th largest into sh.bound, the largest into sh.top. The whole block's.
__device__ __forceinline__ void rank_groups(Shared& sh, float top, int K) {
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (threadIdx.x % 4 == 0) sh.group[threadIdx.x / 4] = top;
  if (threadIdx.x == 0) sh.top = sh.bound = -INFINITY;
  __syncthreads();
  const int mine = threadIdx.x / 4, first = threadIdx.x % 4 * (GROUPS / 4);
  int rank = 0;
#pragma unroll
  for (int j = 0; j < GROUPS / 4; ++j) {
    const float other = sh.group[first + j];
    rank += other > top || (other == top && first + j < mine);
  }
  rank = sum_of_four(rank);
  if (rank == K - 1) sh.bound = top;
  if (rank == 0) sh.top = top;
  __syncthreads();
}

// VALUES: logits a thread has of a tile.
template <int VALUES>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM)
beam_select_kernel(const float* __restrict__ logits, const long long ld, const float* __restrict__ scores, const int V, const int beams, const int K,
                   const int tiles_per_block, float* __restrict__ best, int32_t* __restrict__ parents, int32_t* __restrict__ tokens,
                   Part* __restrict__ parts, Key* __restrict__ lists, int* __restrict__ counters) {
  constexpr int TILE = THREADS * VALUES, STAGE = TILE + 4;
  extern __shared__ __align__(16) float ring[];            // [STAGES][STAGE]
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunk = blockIdx.x, chunks = gridDim.x, item = blockIdx.y / beams;
  const long long row = blockIdx.y;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&sh.full[s]), 1);
    fence_barrier_init();
    fence_proxy_async();
    sh.n = 0;
  }
  __syncthreads();
  gb::pdl_launch_dependents();
  gb::pdl_wait();
  // A stretch of the row: tiles count from the row's first logit, wherever that lies, and a thread has every 256th logit of a tile, so that rows of the same logits
  // have the same sums. (Four neighbouring ones a thread, a load from shared memory instead of four, tie a row's tiles to its place within 16 bytes, and were no faster:
  // 512 rows of 128,256 58.6 and 57.9 us.) Copies are of 16-byte vectors; the row's ends, in front of `head` and from `tail` on, are read where they are used.
  const float* const x_row = logits + row * ld;
  const int shift = (int)((uintptr_t)x_row >> 2 & 3), head = (4 - shift) & 3, tail = V - (V + shift & 3);
  const int tile0 = chunk * tiles_per_block, tiles = min(tiles_per_block, (V + TILE - 1) / TILE - tile0);
  auto place = [&](int tile, int i) { return (tile0 + tile) * TILE + i * THREADS + (int)threadIdx.x; };
  auto fetch = [&](int tile) {           // the vectors that hold the tile's logits
    const int start = (tile0 + tile) * TILE, from = start == 0 ? head : start - shift;
    const int vectors = max(0, min(start + TILE + head, tail) - from) / 4;
    const uint32_t bar = smem_u32(&sh.full[tile % STAGES]);
    if (vectors == 0) {
      mbar_arrive(bar);
      return;
    }
    mbar_arrive_expect_tx(bar, vectors * 16);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(ring + tile % STAGES * STAGE + (from + shift - start))), "l"(x_row + from), "r"(vectors * 16), "r"(bar) : "memory");
  };
  // (the first tiles are asked for before it is known whether the beam is over)
  if (threadIdx.x == 0)
    for (int tile = 0; tile < min(STAGES, tiles); ++tile) fetch(tile);
  if (threadIdx.x < beams) sh.score[threadIdx.x] = scores[(long long)item * beams + threadIdx.x];
  __syncthreads();
  bool ok = true;
  auto gave_up = [&]() {                 // a copy that never came: others in flight need microseconds to land
    gb_err::report(ERR_WAIT_FULL);
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) {}
  };
  if (!is_finite(sh.score[blockIdx.y % beams])) {
    if (threadIdx.x == 0) {
      for (int tile = 0; tile < min(STAGES, tiles); ++tile) ok = mbar_wait(smem_u32(&sh.full[tile]), 0) && ok;
      if (!ok) gave_up();
    }
  } else {
    float x[VALUES];
    auto read = [&](int tile) {
      const float* const from = ring + tile % STAGES * STAGE + shift + threadIdx.x;
      const int start = (tile0 + tile) * TILE;
      if (start >= head && start + TILE <= tail) {
#pragma unroll
        for (int i = 0; i < VALUES; ++i) x[i] = from[i * THREADS];
      } else {
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
          const int at = place(tile, i);
          x[i] = at >= V ? -INFINITY : at >= head && at < tail ? from[i * THREADS] : x_row[at];
        }
      }
    };
    auto largest = [&]() {
      float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
      for (int i = 4; i < VALUES; i += 2) top = fmaxf(top, fmaxf(x[i], x[i + 1]));
      return top;
    };
    float bound = -INFINITY;           // what is no larger is not on the list
    float ref = -INFINITY;             // exponentials are of x - ref, none above e^CLOSE
    double sum = 0.;
    int n = 0, side = 0;               // the list's entries when it was last looked at, and which of the two lists it is
    const int limit = 2 * K + 32;      // entries at which the list is cut
    auto refer_to = [&](float to) {
      if (to > ref + CLOSE) {          // (of the first tile's largest by as much: once or twice a row)
        sum *= exp_of((double)ref - (double)to);
        ref = to;
      }
    };
    // The list becomes its K largest in order (the others behind them, until new ones come). What leaves it goes into the sum, at last all of it.
    auto cut = [&](bool last) {
      const Key* const from = sh.list[side];
      Key* const to = sh.list[side ^ 1];
      for (int i0 = 0; i0 < n; i0 += THREADS / 4) {           // four threads an entry
        const int i = i0 + (int)threadIdx.x / 4;
        const Key mine = i < n ? from[i] : 0;
        int rank = 0;
        for (int j = threadIdx.x % 4; j < n; j += 4) rank += from[j] > mine;
        rank = sum_of_four(rank);
        if (i < n) to[rank] = mine;
      }
      __syncthreads();
      const int kept = min(n, K);
      if (n > 0) {
        refer_to(logit_of(to[0]));
        // (in order: places on the list go to whoever is first)
        for (int i = threadIdx.x; i < n; i += THREADS)
          if (last) sum += exp_of((double)logit_of(to[i]) - (double)ref);
          else if (i >= kept) sum += (double)fast_exp2((logit_of(to[i]) - ref) * 1.4426950408889634f);
        if (kept == K) bound = logit_of(to[kept - 1]);          // (a later logit as large has a larger number)
      }
      side ^= 1;
      n = kept;
      if (threadIdx.x == 0) sh.n = n;
      __syncthreads();
    };
    for (int tile = 0; tile < tiles && ok; ++tile) {
      ok = mbar_wait(smem_u32(&sh.full[tile % STAGES]), tile / STAGES & 1);
      int taken = 0;
      double tile_sum = 0.;
      // those above the bound (and `exactly`) go to the list, the others into the sum; the last place taken
      auto enter = [&](float top, Key exactly) {
        if (top > bound) {
          uint32_t above = 0;
#pragma unroll
          for (int i = 0; i < VALUES; ++i)
            if (x[i] > bound && (exactly == 0 || key_of(x[i], place(tile, i)) >= exactly)) above |= 1u << i, x[i] = -INFINITY;
          while (above) {
            const int i = __ffs(above) - 1, at = place(tile, i);
            above &= above - 1;
            taken = atomicAdd(&sh.n, 1);
            const float value = at >= head && at < tail ? ring[tile % STAGES * STAGE + at + shift - (tile0 + tile) * TILE] : x_row[at];
            if (taken < LIST) sh.list[side][taken] = key_of(value, at);
          }
        }
        // (a multiply-add would round ref log2(e), for all alike)
        const float2 less = ref == -INFINITY ? make_float2(0.f, 0.f) : make_float2(-ref, -ref), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
        float2 rest[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < VALUES; i += 2) {
          const float2 d = mul2(add2(make_float2(x[i], x[i + 1]), less), log2e);
          rest[i >> 1 & 1] = add2(rest[i >> 1 & 1], make_float2(fast_exp2(d.x), fast_exp2(d.y)));
        }
        rest[0] = add2(rest[0], rest[1]);
        tile_sum += (double)(rest[0].x + rest[0].y);
      };
      if (ok) read(tile);
      const float top = largest();
      if (ref == -INFINITY) {          // no logit yet but -inf
        rank_groups(sh, top, K);
        bound = sh.bound == -INFINITY ? -INFINITY : nextafterf(sh.bound, -INFINITY);         // (the bound itself is on the list)
        ref = sh.top;
      }
      enter(top, 0);
      // one barrier a tile: all have read it, and whether the list is long
      const int look = __syncthreads_or(!ok || taken >= limit);
      if (!look) {
        sum += tile_sum;
        if (threadIdx.x == 0 && tile + STAGES < tiles) fetch(tile + STAGES);
        continue;
      }
      ok = __syncthreads_and(ok);
      if (!ok) break;
      n = sh.n;
      if (n <= LIST) {
        sum += tile_sum;
      } else {
        // The list has run over. Out with the tile's entries, and in again by the tile's K-th key, found from its highest bit down: the
        // largest number that K keys are no smaller than.
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < LIST; i += THREADS) {
          const Key k = sh.list[side][i];
          if (index_of(k) < (tile0 + tile) * TILE) sh.list[side ^ 1][atomicAdd(&sh.n, 1)] = k;
        }
        __syncthreads();
        n = sh.n;
        side ^= 1;
        read(tile);
        Key found = 0;
        for (int bit = 63; bit >= 0; --bit) {
          const Key trial = found | (Key)1 << bit;
          int count = 0;
#pragma unroll
          for (int i = 0; i < VALUES; ++i) count += x[i] > bound && key_of(x[i], place(tile, i)) >= trial;
          count = __reduce_add_sync(0xffffffffu, count);
          __syncthreads();
          if (threadIdx.x == 0) sh.n = 0;
          __syncthreads();
          if (lane == 0) atomicAdd(&sh.n, count);
          __syncthreads();
          if (sh.n >= K) found = trial;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.n = n;
        __syncthreads();
        refer_to(logit_of(found));             // (nothing that the tile keeps off the list is larger)
        tile_sum = 0.;
        enter(top, found);
        sum += tile_sum;
        __syncthreads();
        n = sh.n;
      }
      if (threadIdx.x == 0 && tile + STAGES < tiles) fetch(tile + STAGES);
      cut(false);
    }
    __syncthreads();
    n = sh.n;
    __syncthreads();
    if (!ok) {
      if (threadIdx.x == 0) gave_up();
      n = 0, sum = NAN;                  // the stretch counts as no numbers
    }
    cut(true);
    Key* const list = lists + (row * chunks + chunk) * K;
    for (int i = threadIdx.x; i < K; i += THREADS) list[i] = i < n ? sh.list[side][i] : 0;
    sum = warp_sum(sum);
    if (lane == 0) sh.warp[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = warp_sum(lane < WARPS ? sh.warp[lane] : 0.);
      if (lane == 0) parts[row * chunks + chunk] = Part{(double)ref, sum};
    }
  }
  // ---- the item's last block joins the stretches. (The barrier orders the block's writes in front of the count, which is a release, and behind it
  // what the block reads of the others'.)
  __syncthreads();
  if (threadIdx.x == 0) {
    int seen;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counters + item) : "memory");
    sh.last = seen == beams * chunks - 1;
    if (sh.last) counters[item] = 0;              // as the next launch expects it
    sh.n = 0;
  }
  __syncthreads();
  if (!sh.last) return;
  const long long row0 = (long long)item * beams;
  // The entries of all lists, four a thread at a time; the first ones are asked for before the sums are there.
  const int per_row = chunks * K, entries = beams * per_row;          // (chunks: no more than the blocks of a device)
  const Key* const all = lists + row0 * per_row;
  Key mine[4];
  int beam[4];
  auto ask = [&](int e0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = e0 + j * THREADS + threadIdx.x;
      beam[j] = e < entries ? e / per_row : 0;
      mine[j] = e < entries && is_finite(sh.score[beam[j]]) ? __ldcg(all + e) : 0;
    }
  };
  ask(0);
  for (int w = warp; w < beams; w += WARPS) {
    double lse = NAN;
    if (is_finite(sh.score[w])) {
      const Part* const row_parts = parts + (row0 + w) * chunks;
      Part first{-INFINITY, 0.};
      if (lane < chunks) first.ref = __ldcg(&row_parts[lane].ref), first.sum = __ldcg(&row_parts[lane].sum);
      double top = first.ref;
      for (int c = lane + 32; c < chunks; c += 32) top = fmax(top, __ldcg(&row_parts[c].ref));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      double part = first.sum == 0. || first.ref == top ? first.sum : first.sum * exp_of(first.ref - top);
      for (int c = lane + 32; c < chunks; c += 32) part += __ldcg(&row_parts[c].sum) * exp_of(__ldcg(&row_parts[c].ref) - top);
      lse = log(warp_sum(part)) + top;
    }
    if (lane == 0) sh.lse[w] = isfinite(lse) ? lse : NAN;
  }
  __syncthreads();
  Joined& join = *reinterpret_cast<Joined*>(ring);
  auto cut_joined = [&](int n) {                     // becomes its K best in order
    for (int i0 = 0; i0 < n; i0 += THREADS / 4) {
      const int i = i0 + (int)threadIdx.x / 4;
      const Scored mine = i < n ? Scored{join.score[i], join.at[i]} : Scored{INFINITY, -1};
      int rank = 0;
      for (int j = threadIdx.x % 4; j < n; j += 4) rank += in_front(join.score[j], join.at[j], mine.score, mine.at);
      rank = sum_of_four(rank);
      if (rank < K && i < n) sh.won[rank] = mine;
    }
    __syncthreads();
  };
  double least = -INFINITY;                          // what is below is not among the K best
  int n = 0;
  for (int e0 = 0; e0 < entries; e0 += 4 * THREADS) {
    if (e0 > 0) ask(e0);
    double score[4];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      score[j] = mine[j] ? (double)sh.score[beam[j]] + ((double)logit_of(mine[j]) - sh.lse[beam[j]]) : NAN;
      if (score[j] >= least) top = fmaxf(top, __double2float_rd(score[j]));
    }
    if (e0 == 0) {
      rank_groups(sh, top, K);           // as in the rows' first tiles, rounded down
      least = (double)sh.bound;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (score[j] >= least) {                       // (an empty place's is no number)
        const int slot = atomicAdd(&sh.n, 1);
        join.score[slot] = score[j];
        join.at[slot] = (long long)beam[j] * V + index_of(mine[j]);
      }
    __syncthreads();
    n = sh.n;
    if (n > JOINED - 4 * THREADS && e0 + 4 * THREADS < entries) {          // the next ones might not fit
      cut_joined(n);
      n = min(n, K);
      for (int i = threadIdx.x; i < n; i += THREADS) join.score[i] = sh.won[i].score, join.at[i] = sh.won[i].at;
      if (threadIdx.x == 0) sh.n = n;
      if (n == K) least = sh.won[K - 1].score;
    }
    __syncthreads();
  }
  cut_joined(n);
  const int found = min(n, K);
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

// How rows are cut. A small call, of less than a tile of 4,096 an SM, goes by tiles of 1,024. Then as many blocks as run at once, each with its share
// of a row: a block pays for its first bound and its last cut, and the bound rises with the tiles that it has seen. Where there are more rows than that, four
// times as many, so that the last ones do not keep the device waiting. (512 rows of 128,256: a block a row 56 us, two 64, three 70, eight 86; equal stretches, which begin
// and end inside rows, 70: pieces of two rows, and too few registers for what tells them apart.)
struct Cut {
  bool small;
  int per_block, chunks;
};
Cut cut_of(int rows, int V) {
  const long long room = (long long)BLOCKS_PER_SM * gb::sm_count();
  Cut c;
  c.small = (long long)rows * V < (long long)gb::sm_count() * THREADS * MANY;
  const int tile = THREADS * (c.small ? 4 : MANY), tiles = (V + tile - 1) / tile;
  const long long blocks = rows > room ? (4 * room + rows - 1) / rows : room / rows;           // of a row
  c.per_block = (int)((tiles + blocks - 1) / blocks);
  c.chunks = (tiles + c.per_block - 1) / c.per_block;
  return c;
}

}  // namespace

// Bytes of scratch memory of a call, of which the first `counter_bytes` (a counter for every item) are zero before the first one; every call
// leaves them zero.
GB_EXPORT long long gb_beam_select_scratch_bytes(int items, int beams, int V, int K, long long* counter_bytes) {
  const long long rows = (long long)items * beams, chunks = cut_of((int)rows, V).chunks;
  *counter_bytes = ((long long)items * 4 + 15) / 16 * 16;
  return rows * chunks * (long long)(sizeof(Part) + K * sizeof(Key));
}

// What the caller packs, eight bytes each.
struct BeamCall {
  const float *logits, *scores;
  float* best;
  int32_t *parents, *tokens;
  void *counters, *scratch, *stream;
  long long ld, items, beams, V, K;
};
GB_EXPORT int gb_beam_select(const BeamCall* call) {
  const int items = (int)call->items, beams = (int)call->beams, V = (int)call->V, K = (int)call->K;
  if (K > MOST || beams > MOST) return gb::fail(GB_UNSUPPORTED, "beam_select: %d of %d beams (at most %d)", K, beams, MOST);
  const int rows = items * beams;
  if (rows > 65535) return gb::fail(GB_UNSUPPORTED, "beam_select: %d rows of logits", rows);
  const Cut cut = cut_of(rows, V);
  Part* parts = reinterpret_cast<Part*>(call->scratch);
  Key* lists = reinterpret_cast<Key*>(parts + (long long)rows * cut.chunks);
  auto launch = [&](auto values) {
    constexpr int VALUES = decltype(values)::value, RING = STAGES * (THREADS * VALUES + 4) * 4, SMEM = RING > (int)sizeof(Joined) ? RING : (int)sizeof(Joined);
    static gb::OncePerDevice configured;
    if (configured.needed()) {
      const cudaError_t e = cudaFuncSetAttribute(beam_select_kernel<VALUES>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
      if (e != cudaSuccess) return gb::fail(GB_CUDA_ERROR, "beam_select: %s", cudaGetErrorString(e));
      configured.done();
    }
    return gb::check_pdl_launch(gb::launch_pdl(beam_select_kernel<VALUES>, dim3(cut.chunks, rows), dim3(THREADS), SMEM, (cudaStream_t)call->stream, dim3(1),
                                               call->logits, call->ld, call->scores, V, beams, K, cut.per_block, call->best, call->parents, call->tokens, parts,
                                               lists, reinterpret_cast<int*>(call->counters)), "beam_select");
  };
  return cut.small ? launch(std::integral_constant<int, 4>{}) : launch(std::integral_constant<int, MANY>{});
}

GB_EXPORT int gb_beam_select_error_check() { return gb_err::fetch_and_clear(); }
GB_EXPORT int gb_beam_select_set_error_sink(int* host_word) { return gb_err::set_sink(host_word); }
