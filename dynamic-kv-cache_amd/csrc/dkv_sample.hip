// Sampling (gfx950): one token a row from logits and a given random number.
//
// w_i = exp((x_i - max) / temperature); of the tokens in order of their logits (equal ones: the first) the first
// top_k, of those the shortest run that holds top_p of their weight, of those the ones with w >= min_p; then the
// first token, in the vocabulary's order, up to which the kept weight exceeds u times its total.
//
// Weights are computed in 64 bits and summed as integers, multiples of 2^-SHIFT of the largest: such sums are exact
// and the same in every order, so no atomic or split can move a border between two tokens. SHIFT leaves room for
// the sum of a whole vocabulary of weights of one (SHIFT >= 40 up to 4 million tokens; a weight below 2^-41 of the
// largest counts as zero).
#include "dkv_select.h"

namespace dkv {
namespace sample {

constexpr int THREADS = 1024;

struct Row {
  const void* logits;
  int vocab, shift;
  bool bf16;
  float top;           // the largest logit
  double temperature;

  __device__ __forceinline__ float at(int i) const {
    return bf16 ? bf16_lo(static_cast<const uint16_t*>(logits)[i]) : static_cast<const float*>(logits)[i];
  }
  // exp((x - max) / temperature): 0 where x is -infinity or NaN, and beside an infinite logit
  __device__ __forceinline__ double weight(float x) const {
    if (!(x > -INFINITY)) return 0.;
    if (x == top) return 1.;
    return top == INFINITY ? 0. : exp(((double)x - (double)top) / temperature);
  }
  __device__ __forceinline__ uint64_t units(double w) const { return (uint64_t)__builtin_rint(ldexp(w, shift)); }
};

// Tokens of keys above `key`, and of that key up to index `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool takes(uint32_t x, int i) const { return x > key || (x == key && i <= last); }
};

struct Scratch {
  SelectScratch select;
  uint64_t mass[256];
  uint64_t sums[THREADS / 64];
  uint32_t counts[THREADS / 64];
  uint64_t total;
  uint32_t prefix;
  int found;
};

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)x, lane, 64) | (uint64_t)(uint32_t)__shfl((int)(x >> 32), lane, 64) << 32;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t x) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = shfl64(x, (lane - d) & 63);
    if (lane >= d) x += o;
  }
  return x;
}
__device__ __forceinline__ uint64_t block_sum(Scratch& s, uint64_t x) {
  x = wave_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.sums[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t total = 0;
  for (int w = 0; w < THREADS / 64; ++w) total += s.sums[w];
  return total;
}

// The index of the n-th token (n >= 1) with this key, or the last index if there are fewer.
__device__ __forceinline__ int nth_of_key(Scratch& s, const Row& r, uint32_t key, int64_t n) {
  int64_t seen = 0;
  if (threadIdx.x == 0) s.found = r.vocab - 1;
  for (int i0 = 0; i0 < r.vocab; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const bool tie = i < r.vocab && order_key(r.at(i)) == key;
    int count;
    const int64_t rank = seen + block_rank<THREADS>(tie, s.counts, count);
    if (tie && rank == n - 1) s.found = i;
    seen += count;
    if (seen >= n) break;
  }
  __syncthreads();
  return s.found;
}

__global__ __launch_bounds__(THREADS) void sample_kernel(const void* logits, int bf16, int64_t row_stride, int vocab, int shift,
                                                         const void* u, int u_dtype, dkv_sampling p, int64_t* out) {
  __shared__ Scratch s;
  const int row = blockIdx.x;
  Row r;
  r.bf16 = bf16, r.vocab = vocab, r.shift = shift;
  r.logits = bf16 ? (const void*)(static_cast<const uint16_t*>(logits) + row * row_stride)
                  : (const void*)(static_cast<const float*>(logits) + row * row_stride);
  r.temperature = p.temperature_rows ? (double)p.temperature_rows[row] : p.temperature;
  const int64_t top_k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
  const double top_p = p.top_p_rows ? (double)p.top_p_rows[row] : p.top_p;
  const double min_p = p.min_p_rows ? (double)p.min_p_rows[row] : p.min_p;

  uint32_t best = 0;
  for (int i = threadIdx.x; i < vocab; i += THREADS) best = max(best, order_key(r.at(i)));
#pragma unroll
  for (int d = 32; d; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d, 64));
  if ((threadIdx.x & 63) == 0) s.counts[threadIdx.x >> 6] = best;
  __syncthreads();
  for (int w = 0; w < THREADS / 64; ++w) best = max(best, s.counts[w]);
  __syncthreads();
  if (best <= order_key(-INFINITY)) {  // no token can be drawn
    if (threadIdx.x == 0) out[row] = -1;
    return;
  }
  if (!(r.temperature > 0.)) {
    const int first = nth_of_key(s, r, best, 1);
    if (threadIdx.x == 0) out[row] = first;
    return;
  }
  r.top = __uint_as_float(best & 0x80000000u ? best & 0x7fffffffu : ~best);

  Cut ranked{0, vocab};
  if (top_k > 0 && top_k < vocab) {
    int ties;
    ranked.key = kth_largest<THREADS>(s.select, vocab, (uint32_t)top_k, ties, [&](int i, uint32_t& x) {
      x = order_key(r.at(i));
      return true;
    });
    ranked.last = nth_of_key(s, r, ranked.key, ties);
  }
  Cut held{0, vocab};
  if (top_p < 1.) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
      const float x = r.at(i);
      if (ranked.takes(order_key(x), i)) mine += r.units(r.weight(x));
    }
    // kept while the weight before a token is below this
    uint64_t need = (uint64_t)ceil(fmax(top_p, 0.) * (double)block_sum(s, mine));
    if (need == 0) need = 1;
    uint32_t prefix = 0;
    for (int at = 24; at >= 0; at -= 8) {  // the digit in which the weight from the top reaches it
      for (int i = threadIdx.x; i < 256; i += THREADS) s.mass[i] = 0;
      __syncthreads();
      const uint32_t above = at == 24 ? 0u : ~0u << (at + 8);
      for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float x = r.at(i);
        const uint32_t key = order_key(x);
        if ((key & above) == prefix && ranked.takes(key, i))
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[(key >> at) & 255u]), (unsigned long long)r.units(r.weight(x)));
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int d = 255;
        uint64_t left = need;
        while (d > 0 && s.mass[d] < left) left -= s.mass[d--];
        s.prefix = prefix | (uint32_t)d << at;
        s.total = left;
      }
      __syncthreads();
      prefix = s.prefix, need = s.total;
    }
    held.key = prefix;
    const uint64_t each = r.units(r.weight(__uint_as_float(prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix)));
    held.last = nth_of_key(s, r, prefix, each ? (int64_t)((need + each - 1) / each) : vocab);
  }

  // Each wave takes a consecutive part of the vocabulary; the one in which the weight exceeds the target finds where.
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = (vocab + THREADS / 64 - 1) / (THREADS / 64);
  const int from = wave * part, to = min(vocab, from + part);
  auto kept = [&](int i) -> uint64_t {
    if (i >= to) return 0;
    const float x = r.at(i);
    const uint32_t key = order_key(x);
    if (!ranked.takes(key, i) || !held.takes(key, i)) return 0;
    const double w = r.weight(x);
    return w >= min_p ? r.units(w) : 0;
  };
  uint64_t mine = 0;
  for (int i = from + lane; i < to; i += 64) mine += kept(i);
  const uint64_t total = block_sum(s, mine);
  const double v = u_dtype ? static_cast<const double*>(u)[row] : (double)static_cast<const float*>(u)[row];
  uint64_t target = (uint64_t)(fmin(fmax(v, 0.), 1.) * (double)total);
  if (target >= total) target = total - 1;  // u of one, or rounded up to it: the last kept token
  uint64_t before = 0;
  for (int w = 0; w < wave; ++w) before += s.sums[w];
  if (target < before || target >= before + s.sums[wave]) return;
  for (int i0 = from; i0 < to; i0 += 64) {
    const uint64_t sum = before + wave_scan(kept(i0 + lane));
    const uint64_t over = __ballot(sum > target);
    if (over) {
      if (lane == 0) out[row] = i0 + __ffsll((unsigned long long)over) - 1;
      return;
    }
    before = shfl64(sum, 63);
  }
}

}  // namespace sample
}  // namespace dkv

using namespace dkv;

extern "C" int dkv_sample(const void* logits, int32_t dtype, int64_t row_stride, int32_t rows, int32_t vocab, const void* u,
                          int32_t u_dtype, const dkv_sampling* sampling, int64_t* out, void* stream) {
  clear_error();
  if (!sampling || rows < 0 || vocab <= 0 || row_stride < 0 || dtype < 0 || dtype > 1 || u_dtype < 0 || u_dtype > 1) {
    set_error("dkv_sample: bad arguments (rows %d, vocab %d; logits bf16 (0) or fp32 (1), u fp32 (0) or fp64 (1))", rows, vocab);
    return DKV_EINVAL;
  }
  if (vocab > 1 << 22) {
    set_error("dkv_sample: at most %d tokens in a vocabulary, got %d", 1 << 22, vocab);
    return DKV_EINVAL;
  }
  const dkv_sampling& p = *sampling;
  if ((!p.temperature_rows && !(p.temperature >= 0.)) || (!p.top_k_rows && p.top_k < 0) ||
      (!p.top_p_rows && !(p.top_p > 0. && p.top_p <= 1.)) || (!p.min_p_rows && !(p.min_p >= 0. && p.min_p <= 1.))) {
    set_error("dkv_sample: temperature %g and top_k %d must not be negative, top_p %g in (0, 1], min_p %g in [0, 1]",
              p.temperature, p.top_k, p.top_p, p.min_p);
    return DKV_EINVAL;
  }
  if (rows == 0) return 0;
  if (!logits || !u || !out) {
    set_error("dkv_sample: null pointer argument");
    return DKV_EINVAL;
  }
  int shift = 62;
  while (shift > 62 - 1 || ((uint64_t)vocab >> (62 - shift)) > 0) --shift;  // vocab << shift stays below 2^62
  shift = shift > 52 ? 52 : shift;
  hipLaunchKernelGGL(sample::sample_kernel, dim3(rows), dim3(sample::THREADS), 0, (hipStream_t)stream, logits, dtype == 0, row_stride,
                     vocab, shift, u, u_dtype, p, out);
  return (int)hipGetLastError();
}
