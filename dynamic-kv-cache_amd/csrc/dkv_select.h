// The k largest of n keys by one workgroup, in order: a radix search for the k-th largest key over counts in LDS, from
// the first bit in which the keys differ down to a digit's value that at most 64 keys have, which a wave ranks; then
// each wave takes what it has from its own stretch of the elements. Exact, and the same whatever the order of the
// atomics.
#pragma once
#include "dkv_common.h"

namespace dkv {

// fp32 as an unsigned key of the same order: -0 and +0 are equal, NaN comes before every number.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Counts of a digit's values, in copies by lane: keys of one exponent meet in few bins.
template <int THREADS, int BITS>
struct SelectScratch {
  static constexpr int BINS = 1 << BITS, COPIES = 4;
  uint32_t count[COPIES][BINS];
  uint32_t sums[THREADS / 64], high[THREADS / 64], low[THREADS / 64], few[64];
  uint32_t prefix, left, held, listed;
  int above[THREADS / 64], ties[THREADS / 64];
};

// each(f) calls f(key) for this thread's keys. Returns the k-th largest key of the workgroup (which has at least k of
// them, k >= 1) and in `ties` how many elements of exactly that key belong to the k. All threads call it.
template <int THREADS, int BITS, class Each>
__device__ __forceinline__ uint32_t kth_largest(SelectScratch<THREADS, BITS>& s, uint32_t k, int& ties, Each each) {
  constexpr int BINS = 1 << BITS, COPIES = SelectScratch<THREADS, BITS>::COPIES;
  constexpr int MINE = BINS > THREADS ? BINS / THREADS : 1;  // bins a thread sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t high = 0, low = ~0u;
  each([&](uint32_t x) { high = max(high, x), low = min(low, x); });
#pragma unroll
  for (int d = 32; d; d >>= 1) high = max(high, (uint32_t)__shfl_xor((int)high, d, 64)), low = min(low, (uint32_t)__shfl_xor((int)low, d, 64));
  __syncthreads();
  if (lane == 0) s.high[wave] = high, s.low[wave] = low;
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) high = max(high, s.high[w]), low = min(low, s.low[w]);
  int top = 32 - __clz((int)(high ^ low));           // bits not known yet (32 - clz(0) = 0: all are equal)
  uint32_t known = top == 32 ? 0u : ~0u << top, prefix = high & known;  // the bits found, and which
  while (top > 0) {
    const int shift = max(top - BITS, 0);
    const uint32_t digits = (1u << (top - shift)) - 1;
    for (int i = threadIdx.x; i < COPIES * BINS; i += THREADS) (&s.count[0][0])[i] = 0;
    __syncthreads();
    each([&](uint32_t x) {
      if ((x & known) == prefix) atomicAdd(&s.count[lane % COPIES][(x >> shift) & digits], 1u);
    });
    __syncthreads();
    // thread t has bins from the top: BINS - 1 - t * MINE down
    uint32_t c[MINE], sum = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int bin = BINS - 1 - (int)threadIdx.x * MINE - i;
      c[i] = 0;
#pragma unroll
      for (int j = 0; j < COPIES; ++j) c[i] += bin >= 0 ? s.count[j][bin] : 0u;
      sum += c[i];
    }
    uint32_t upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    if (lane == 63) s.sums[wave] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) upto += w < wave ? s.sums[w] : 0;
    uint32_t higher = upto - sum;
    if (higher < k && k <= upto) {  // one thread
      int i = 0;
#pragma unroll
      for (int j = 0; j + 1 < MINE; ++j)
        if (i == j && higher + c[j] < k) higher += c[j], i = j + 1;
      s.prefix = prefix | (uint32_t)(BINS - 1 - (int)threadIdx.x * MINE - i) << shift;
      s.left = k - higher;
#pragma unroll
      for (int j = 0; j < MINE; ++j)
        if (i == j) s.held = c[j];
    }
    __syncthreads();
    prefix = s.prefix, k = s.left;
    known |= digits << shift, top = shift;
    if (top > 0 && s.held <= 64) {
      each([&](uint32_t x) {
        if ((x & known) == prefix) s.few[atomicAdd(&s.listed, 1u)] = x;
      });
      __syncthreads();
      if (wave == 0) {
        const uint32_t n = s.listed, mine = s.few[lane];
        uint32_t before = 0, same = 0;
        for (uint32_t j = 0; j < n; ++j) {
          const uint32_t x = s.few[j];
          before += x > mine, same += x == mine;
        }
        if ((uint32_t)lane < n && before < k && k <= before + same) s.prefix = mine, s.left = k - before;  // (equal lanes alike)
      }
      __syncthreads();
      prefix = s.prefix, k = s.left;
      break;
    }
  }
  ties = (int)k;
  return prefix;
}

__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Elements [0, n) of a workgroup, a consecutive stretch a wave; up to 64 * N of a wave's keys stay in registers (N = 0:
// none do, and they are loaded again each time). load(i) gives element i's key, 0 where it takes no part.
template <int THREADS, int N, class Load>
struct Elements {
  static constexpr int AHEAD = 8;  // loads in flight
  Load load;
  int n, from, to;
  uint32_t x[N ? N : 1];

  __device__ __forceinline__ Elements(int n_, Load load_) : load(load_), n(n_) {
    const int span = ((n + THREADS / 64 - 1) / (THREADS / 64) + 63) & ~63;
    from = min(n, (int)(threadIdx.x >> 6) * span), to = min(n, from + span);
    if (N) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = from + 64 * j + (int)(threadIdx.x & 63);
        const uint32_t key = load(min(i, n - 1));  // (without a branch: the loads are in flight together)
        x[j] = i < to ? key : 0u;
      }
    }
  }
  // f(i, key) for all lanes together, key 0 past the end
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 63;
    if (N) {
#pragma unroll
      for (int j = 0; j < N; ++j) f(from + 64 * j + lane, x[j]);
    } else {
      for (int i0 = from; i0 < to; i0 += 64 * AHEAD) {
        uint32_t y[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int i = i0 + 64 * j + lane;
          const uint32_t key = load(min(i, n - 1));
          y[j] = i < to ? key : 0u;
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (i0 + 64 * j < to) f(i0 + 64 * j + lane, y[j]);
      }
    }
  }
  // The k largest (equal keys: the first elements): take(place, i) for each, in order, places from 0 on.
  template <int BITS, class Take>
  __device__ __forceinline__ void largest(SelectScratch<THREADS, BITS>& s, uint32_t k, Take take) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int ties;
    const uint32_t at = __builtin_amdgcn_readfirstlane(kth_largest<THREADS, BITS>(s, k, ties, [&](auto f) {
      each([&](int, uint32_t key) {
        if (key) f(key);
      });
    }));
    int above = 0, tied = 0;
    each([&](int, uint32_t key) {
      above += __popcll(__ballot(key > at));
      tied += __popcll(__ballot(key == at));
    });
    uint32_t again = at;  // (opaque: the ballots are taken again below, not held in scalar registers until then)
    asm volatile("" : "+s"(again));
    if (lane == 0) s.above[wave] = above, s.ties[wave] = tied;
    __syncthreads();
    above = tied = 0;  // of the waves before
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w)
      if (w < wave) above += s.above[w], tied += s.ties[w];
    each([&](int i, uint32_t key) {
      const uint64_t more = __ballot(key > again), same = __ballot(key == again);
      const int rank = tied + lanes_before(same);
      if (key > again || (key == again && rank < ties)) take(above + lanes_before(more) + min(rank, ties), i);
      above += __popcll(more), tied += __popcll(same);
    });
  }
};

// Exclusive rank of this thread among those of the workgroup with `flag`, in thread order; `total` gets
// their number. `sums` holds one value a wave; a barrier comes first and last.
template <int THREADS>
__device__ __forceinline__ int block_rank(bool flag, uint32_t (&sums)[THREADS / 64], int& total) {
  const uint64_t b = __ballot(flag);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();
  if (lane == 0) sums[wave] = __popcll(b);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before + lanes_before(b);
}

}  // namespace dkv
