// The k largest of n keys by one workgroup: a radix search for the k-th largest key, eight bits a pass
// from the top, over counts in LDS. Exact, and the same whatever the order of the atomics.
#pragma once
#include "dkv_common.h"

namespace dkv {

// fp32 as an unsigned key of the same order: -0 and +0 are equal, NaN comes before every number.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectScratch {
  uint32_t count[256];
  uint32_t prefix, left;
};

// key(i, x) says whether element i takes part and gives its key in x. Returns the k-th largest key among
// those that do (at least k of them, k >= 1) and in `ties` how many elements of exactly that key belong to
// the k. All threads of the workgroup call it; `s` can be used again after a barrier.
template <int THREADS, class Key>
__device__ __forceinline__ uint32_t kth_largest(SelectScratch& s, int n, uint32_t k, int& ties, Key key) {
  uint32_t prefix = 0;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += THREADS) s.count[i] = 0;
    __syncthreads();
    const uint32_t above = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = threadIdx.x; i < n; i += THREADS) {
      uint32_t x;
      if (key(i, x) && (x & above) == prefix) atomicAdd(&s.count[(x >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // lane l: digits [4 l, 4 l + 4), summed from the top
      uint32_t c[4], sum = 0;
      for (int i = 0; i < 4; ++i) sum += c[i] = s.count[4 * threadIdx.x + i];
      uint32_t from = sum;  // elements whose digit is in this lane's four or a higher lane's
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_down(from, d, 64);
        if (threadIdx.x + d < 64) from += o;
      }
      uint32_t higher = from - sum;
      if (higher < k && k <= from) {  // one lane
        int i = 3;
        while (i > 0 && higher + c[i] < k) higher += c[i--];
        s.prefix = prefix | (4 * threadIdx.x + i) << shift;
        s.left = k - higher;
      }
    }
    __syncthreads();
    prefix = s.prefix;
    k = s.left;
  }
  ties = (int)k;
  return prefix;
}

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
  return before + __popcll(b & ((1ull << lane) - 1));
}

}  // namespace dkv
