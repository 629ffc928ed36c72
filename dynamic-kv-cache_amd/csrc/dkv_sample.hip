// Sampling (gfx950): one token a row from logits and a given random number.
//
// w_i = exp((x_i - max) / temperature); of the tokens in order of their logits (equal ones: the first) the first
// top_k, of those the shortest run that holds top_p of their weight, of those the ones with w >= min_p; then the
// first token, in the vocabulary's order, up to which the kept weight exceeds u times its total.
//
// Weights are computed in 64 bits and summed as integers, multiples of a unit: 2^-SHIFT of a power of two above the row's
// largest weight, at most twice that weight. Integer sums are the same in every order, so no order of the atomics moves a
// border between two tokens. SHIFT leaves room for a whole vocabulary's sum (40 for 4 million tokens, 46 for 49280); what
// is lighter counts as nothing. A weight is rounded to the unit of its part, which may be finer than the row's, and a
// part's sums by bins (at most 401) to the row's when they are joined, down each time. So a border lies less than
// vocab + 401 * parts units from where exact sums have it (1.7e-9 of the largest weight at 49280 tokens in 25 parts), and
// as the parts follow from the number of rows, a row whose random number is as near to a border as that may give the
// neighbouring token in a batch of another size.
//
// weigh_kernel: many workgroups a row, each over a part of the vocabulary, sum its weights by bins, eight an octave, so
// that a bin's tokens are consecutive in the order of the logits. A workgroup alone gets some 30 GB/s from memory that
// others wrote, so no workgroup reads a whole row again:
//   - with a top_k up to SMALL_K, weigh_kernel lists what its part can have among the row's first top_k, and
//     draw_kernel, a workgroup a row, works on these lists alone: two launches;
//   - else pick_kernel joins a row's bins and finds the first one that a filter cuts, gather_kernel lists that bin's
//     tokens, and draw_kernel ranks them and finds the part and the token where the kept weight passes the target.
// Measured: one row of 49280 bf16 logits with top_k 50 and top_p 22.3 us a call (10.9 + 12.7: latency, the lists' ranking and
// four scans); 128 rows of 128003 fp32 logits with top_p and min_p 69.5 (29.2: an exponential in 64 bits and an LDS
// atomic a logit, 65.5 MB at 2.2 TB/s; 7.0; 16.8: the logits again, 3.9 TB/s; 20.4).
// What does not fit that (an infinite logit, exponents beyond 65536, more tokens in a list than it holds) takes
// search_row, a radix search over the whole row, in draw_kernel.
#include "dkv_select.h"

namespace dkv {
namespace sample {

constexpr int THREADS = 512;

template <class T>  // uint16_t: bf16
struct Row {
  const T* logits;
  int vocab, shift;
  float top;           // the largest logit
  double temperature;

  __device__ __forceinline__ float at(int i) const { return value(logits[i]); }
  __device__ __forceinline__ static float value(uint16_t x) { return bf16_lo(x); }
  __device__ __forceinline__ static float value(float x) { return x; }
  // Calls f(token, logit) for tokens first + j * STEP below `end`, N loads in flight.
  template <int N, int STEP, class F>
  __device__ __forceinline__ void each(int first, int end, F f) const {
    for (int i = first; i < end; i += N * STEP) {
      T x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = logits[min(i + j * STEP, end - 1)];
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (i + j * STEP < end) f(i + j * STEP, value(x[j]));
    }
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
  SelectScratch<THREADS, 8> select;
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
template <class T>
__device__ __forceinline__ int nth_of_key(Scratch& s, const Row<T>& r, uint32_t key, int64_t n) {
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

struct Filters {
  double temperature, top_p, min_p, u;
  int64_t top_k;
};

struct Args {
  const void* logits;
  const void* u;
  int64_t row_stride;
  int64_t* out;
  int vocab, shift, u_dtype;
  int parts, part_len;  // of the vocabulary
  int counting;         // a top_k may be set: weigh_kernel counts, too
  dkv_sampling p;
};

template <class T>
__device__ __forceinline__ Row<T> row_of(const Args& a, int row) {
  Row<T> r;
  r.vocab = a.vocab, r.shift = a.shift, r.top = 0.f;
  r.logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  r.temperature = a.p.temperature_rows ? (double)a.p.temperature_rows[row] : a.p.temperature;
  return r;
}

__device__ __forceinline__ Filters filters_of(const Args& a, int row) {
  Filters f;
  f.top_k = a.p.top_k_rows ? a.p.top_k_rows[row] : a.p.top_k;
  f.top_p = a.p.top_p_rows ? (double)a.p.top_p_rows[row] : a.p.top_p;
  f.min_p = a.p.min_p_rows ? fmin((double)a.p.min_p_rows[row], 1.) : a.p.min_p;
  const double u = a.u_dtype ? static_cast<const double*>(a.u)[row] : (double)static_cast<const float*>(a.u)[row];
  f.u = fmin(fmax(u, 0.), 1.);
  return f;
}

__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// floor(p * total), or ceil where `up`, exactly: a total has more bits than a double. p in [0, 1].
__device__ __forceinline__ uint64_t share_of(double p, uint64_t total, bool up) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  if (!(p > 1e-300)) return up && p > 0. ? 1 : 0;
  const uint64_t m = (bits & ((1ull << 52) - 1)) | 1ull << 52;
  const int k = 1075 - (int)(bits >> 52);  // p = m / 2^k, k >= 52
  const uint64_t high = __umul64hi(m, total), low = m * total;
  if (k >= 128) return up ? 1 : 0;
  const uint64_t floor_ = k >= 64 ? (k == 64 ? high : high >> (k - 64)) : high << (64 - k) | low >> k;
  const bool rest = k >= 64 ? low || (k > 64 && (high & ((1ull << (k - 64)) - 1))) : low & ((1ull << k) - 1);
  return floor_ + (up && rest ? 1 : 0);
}

// The kept weight's unit in which the token lies (u of one: the last).
__device__ __forceinline__ uint64_t target_of(double u, uint64_t total) {
  const uint64_t target = share_of(u, total, false);
  return target >= total ? total - 1 : target;
}

// The whole row by radix searches: right for every row, and slow (every search reads all of it).
template <class T>
__device__ __forceinline__ void search_row(Scratch& s, const Row<T>& r, const Filters& f, int64_t* out) {
  const int vocab = r.vocab;
  const int64_t top_k = f.top_k;
  const double top_p = f.top_p, min_p = f.min_p;
  Cut ranked{0, vocab};
  if (top_k > 0 && top_k < vocab) {
    int ties;
    ranked.key = kth_largest<THREADS, 8>(s.select, (uint32_t)top_k, ties, [&](auto f) {
      for (int i = threadIdx.x; i < vocab; i += THREADS) f(order_key(r.at(i)));
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
    uint64_t need = share_of(fmax(top_p, 0.), block_sum(s, mine), true);
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
    const uint64_t each = r.units(r.weight(logit_of(prefix)));
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
  const uint64_t target = target_of(f.u, total);
  uint64_t before = 0;
  for (int w = 0; w < wave; ++w) before += s.sums[w];
  if (target < before || target >= before + s.sums[wave]) return;
  for (int i0 = from; i0 < to; i0 += 64) {
    const uint64_t sum = before + wave_scan(kept(i0 + lane));
    const uint64_t over = __ballot(sum > target);
    if (over) {
      if (lane == 0) *out = i0 + __ffsll((unsigned long long)over) - 1;
      return;
    }
    before = shfl64(sum, 63);
  }
}

// ---- bins -------------------------------------------------------------------------------------------------------
constexpr int WEIGH_THREADS = 256;
constexpr int HELD = 32;               // tokens a thread of weigh_kernel keeps in registers, where a part is that small
constexpr int OCTAVE = 8, BINS = 512;  // bins of an octave of weight; at most 8 * 50 + 1 are used
constexpr int STEPS = 256;             // steps of the table of 2^f
constexpr int SUBS = STEPS / OCTAVE;   // of them in a bin
constexpr int LIST = 4096;             // tokens of a bin that is cut
// top_k whose tokens are listed by the parts: one row of 49280 bf16 logits 26.8 us at 100 and 39.9 at 250 against 50.4 by
// bins, 128 rows of 128003 fp32 logits 58.7 and 74.8 against 101.
constexpr int SMALL_K = 256;
constexpr int PART_LIST = 512;         // tokens that a part lists
constexpr int MAX_PARTS = 64;
constexpr int ROWS = 512;              // rows of one set of launches
constexpr int AHEAD = 8;               // parts whose bins a thread has in flight
constexpr int NOTHING = INT32_MIN, BEYOND = INT32_MAX;
constexpr double FAR = 65536.;         // largest exponent whose weights keep 2^-36 of their value
constexpr double LOG2_E = 1.44269504088896340736, LN_2 = 0.69314718055994530942;

struct Part {
  float top;     // its largest logit, and at temperature 0 the first index of it
  int first;
  int exponent;  // its weights are below 2^(exponent + 1): the unit of its sums is 2^(exponent - SHIFT)
  int listed;    // tokens in its list
};

struct RowState {
  float top;
  int exponent, bin;    // the row's exponent; the first bin that a filter cuts (BINS: none)
  uint32_t low, high;   // keys of that bin
  int listed;           // of its tokens, in the row's list
  int search;           // takes search_row
  int pad;
};

struct Work {
  uint64_t* masses;    // [parts][BINS]
  uint64_t* part_list;  // [parts][PART_LIST] tokens: ~key << 32 | index
  uint64_t* sums;      // [rows][BINS] weight from the top bin on
  uint64_t* lists;     // [rows][LIST] tokens
  Part* parts;
  RowState* rows;
  uint32_t* counts;    // [parts][BINS]
  uint32_t* count_sums;  // [rows][BINS]
};

__device__ __forceinline__ bool lists_parts(const Filters& f) { return f.top_k > 0 && f.top_k <= SMALL_K; }

__device__ __forceinline__ uint64_t token_of(uint32_t key, int index) { return (uint64_t)~key << 32 | (uint32_t)index; }
__device__ __forceinline__ uint32_t key_of(uint64_t token) { return ~(uint32_t)(token >> 32); }
__device__ __forceinline__ int index_of(uint64_t token) { return (int)(uint32_t)token; }

// Weights relative to 2^exponent. Y = x log2(e) / T is rounded to a multiple k of 1/256 by an addition that leaves k in
// the sum's low bits; 2^Y is a table's 2^((k mod 256) / 256) times the exponential series of the rest (at most
// ln 2 / 512, so the fifth term is below 2^-53).
struct Weigher {
  const double* table;
  double rate;  // log2(e) / T
  int shift, exponent;
  float least;  // weights of smaller logits are nothing

  __device__ __forceinline__ Weigher(const double* table_, double temperature, int shift_, int exponent_)
      : table(table_), rate(LOG2_E / temperature), shift(shift_), exponent(exponent_) {
    least = fmaxf((float)((exponent - shift - 2) / rate), -3.4028235e38f);
  }
  __device__ __forceinline__ static double magic() { return 1.5 * (1ll << 44); }
  __device__ __forceinline__ int step(float x) const {
    return (int)(uint32_t)__builtin_bit_cast(uint64_t, (double)x * rate + magic());
  }
  // The weight in units of 2^(exponent - shift), rounded down, and its bin from 8 * exponent down.
  __device__ __forceinline__ uint64_t weight(float x, int& bin) const {
    bin = BINS;
    if (!(x >= least)) return 0;
    const double y = (double)x * rate, sum = y + magic(), r = y - (sum - magic());
    const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, sum), down = exponent - (k >> 8);
    double e = __builtin_fma(r, LN_2 * LN_2 * LN_2 * LN_2 / 24, LN_2 * LN_2 * LN_2 / 6);
    e = __builtin_fma(r, e, LN_2 * LN_2 / 2);
    e = __builtin_fma(r, e, LN_2);
    const double t = table[k & (STEPS - 1)], w = __builtin_fma(t, r * e, t);
    if (down > shift) return 0;
    bin = OCTAVE * exponent - (k >> 5);
    // w 2^51 as the low bits of a sum with 2^52
    const uint64_t m = __builtin_bit_cast(uint64_t, __builtin_fma(w, 0x1p51, 0x1p52)) & ((1ull << 52) - 1);
    return m >> (51 - shift + down);
  }
  __device__ __forceinline__ uint64_t weight(float x) const {
    int bin;
    return weight(x, bin);
  }
  // The smallest key whose step is `first` or more, by weight()'s own arithmetic. The border is half a step below; a
  // float that near it is at most a few keys off.
  __device__ __forceinline__ uint32_t first_key(int first) const {
    const float x = (float)((first - .5) / STEPS / rate);
    uint32_t key = order_key(fminf(fmaxf(x, -3.4028235e38f), 3.4028235e38f));
    auto reaches = [&](uint32_t k) { return step(logit_of(k)) >= first; };
    for (int i = 0; i < 8 && reaches(key - 1); ++i) --key;
    for (int i = 0; i < 8 && !reaches(key); ++i) ++key;
    return key;
  }
  // The smallest step of a bin.
  __device__ __forceinline__ int bin_step(int bin) const { return SUBS * (OCTAVE * exponent - bin); }
};

template <class T>
__global__ __launch_bounds__(WEIGH_THREADS) void weigh_kernel(Args a, Work work) {
  __shared__ double table[STEPS];
  __shared__ uint64_t mass[BINS];
  __shared__ uint32_t count[BINS];
  __shared__ float best[WEIGH_THREADS / 64];
  __shared__ int at[WEIGH_THREADS / 64];
  __shared__ int listed, last_bin;
  const int part = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Row<T> r = row_of<T>(a, row);
  const Filters f = filters_of(a, row);
  const int from = part * a.part_len, to = min(a.vocab, from + a.part_len);
  const int64_t slot = (int64_t)row * a.parts + part;
  const bool fits = a.part_len <= HELD * WEIGH_THREADS;
  float held[HELD];
  if (fits && from < to) {
    T x[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) x[j] = r.logits[min(from + j * WEIGH_THREADS + (int)threadIdx.x, to - 1)];
#pragma unroll
    for (int j = 0; j < HELD; ++j) held[j] = Row<T>::value(x[j]);
  }
  auto each = [&](auto g) {  // g(token, logit) for this thread's tokens
    if (fits) {
#pragma unroll
      for (int j = 0; j < HELD; ++j)
        if (const int i = from + j * WEIGH_THREADS + (int)threadIdx.x; i < to) g(i, held[j]);
    } else {
      r.template each<8, WEIGH_THREADS>(from + threadIdx.x, to, g);
    }
  };
  for (int i = threadIdx.x; i < STEPS; i += WEIGH_THREADS) table[i] = exp2(i * (1. / STEPS));
  for (int i = threadIdx.x; i < BINS; i += WEIGH_THREADS) mass[i] = 0, count[i] = 0;
  if (threadIdx.x == 0) listed = 0, last_bin = BINS;
  float top = -INFINITY;
  each([&](int, float x) { top = fmaxf(top, x); });  // (passes over NaN)
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
  if (lane == 0) best[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WEIGH_THREADS / 64; ++w) top = fmaxf(top, best[w]);
  if (!(r.temperature > 0.)) {
    int first = to;
    each([&](int i, float x) {
      if (x == top) first = min(first, i);
    });
#pragma unroll
    for (int d = 32; d; d >>= 1) first = min(first, __shfl_xor(first, d, 64));
    if (lane == 0) at[wave] = first;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 0; w < WEIGH_THREADS / 64; ++w) first = min(first, at[w]);
      work.parts[slot] = Part{top, first, top > -INFINITY ? 0 : NOTHING, 0};
    }
    return;
  }
  const double y = (double)top * (LOG2_E / r.temperature);
  // (a part far below the others, of masked tokens say, just adds nothing)
  const int exponent = !(top > -INFINITY) ? NOTHING : top < INFINITY && y <= FAR ? (int)fmax(floor(y) + 1., -1e9) : BEYOND;
  const bool far = exponent == NOTHING || exponent == BEYOND || exponent < -FAR - BINS;  // (a row below -FAR is searched)
  if (threadIdx.x == 0 && (far || !lists_parts(f))) work.parts[slot] = Part{top, 0, exponent, 0};
  if (far) return;
  const Weigher weigher(table, r.temperature, a.shift, exponent);
  const bool lists = lists_parts(f);
  each([&](int, float x) {
    int bin;
    const uint64_t w = weigher.weight(x, bin);
    if (w) {
      if (!lists) atomicAdd(reinterpret_cast<unsigned long long*>(&mass[bin]), (unsigned long long)w);
      if (a.counting) atomicAdd(&count[bin], 1u);
    }
  });
  __syncthreads();
  if (!lists) {
    for (int i = threadIdx.x; i <= OCTAVE * a.shift; i += WEIGH_THREADS) {
      work.masses[slot * BINS + i] = mass[i];
      if (a.counting) work.counts[slot * BINS + i] = count[i];
    }
    return;
  }
  // tokens down to the bin in which the part's count reaches top_k
  if (wave == 0) {
    uint32_t c[BINS / 64], sum = 0;
#pragma unroll
    for (int i = 0; i < BINS / 64; ++i) sum += c[i] = count[lane * (BINS / 64) + i];
    uint32_t upto = sum;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    uint32_t before = upto - sum;
    if (before < f.top_k && f.top_k <= upto) {
      int i = 0;
      while (before + c[i] < f.top_k) before += c[i++];
      last_bin = lane * (BINS / 64) + i;
    }
  }
  __syncthreads();
  const int last = last_bin;
  each([&](int i, float x) {
    int bin;
    if (x >= weigher.least && OCTAVE * exponent - (weigher.step(x) >> 5) <= last && weigher.weight(x, bin)) {
      const int to = atomicAdd(&listed, 1);
      if (to < PART_LIST) work.part_list[slot * PART_LIST + to] = token_of(order_key(x), i);
    }
  });
  __syncthreads();
  if (threadIdx.x == 0) work.parts[slot] = Part{top, 0, exponent, listed};
}

struct RowTop {
  float top;
  int first, exponent;
};
// The row's largest logit, its first index (temperature 0) and exponent, by every wave from its parts: lane p has part p
// (MAX_PARTS is a wave).
__device__ __forceinline__ RowTop row_top(const Part& mine) {
  RowTop t{mine.top, mine.first, mine.exponent};
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float top = __shfl_xor(t.top, d, 64);
    const int first = __shfl_xor(t.first, d, 64), exponent = __shfl_xor(t.exponent, d, 64);
    if (top > t.top || (top == t.top && first < t.first)) t.top = top, t.first = first;
    t.exponent = max(t.exponent, exponent);
  }
  return t;
}
__device__ __forceinline__ Part part_of(const Args& a, const Part* parts, int lane) {
  return lane < a.parts ? parts[lane] : Part{-INFINITY, a.vocab, NOTHING, 0};
}
// Octaves from the row's exponent down to a part's (more than any weight has where the part has none).
__device__ __forceinline__ int apart_of(int row_exponent, int exponent) {
  return exponent == NOTHING ? BINS : (int)min((int64_t)row_exponent - exponent, (int64_t)BINS);
}

struct BinScratch {
  uint64_t sums[THREADS / 64];
  uint64_t before;
  int bin;
};

template <int WAVES>
__device__ __forceinline__ uint64_t block_scan(uint64_t (&sums)[THREADS / 64], uint64_t x, uint64_t& total) {  // inclusive
  x = wave_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += sums[w];
    total += sums[w];
  }
  return before + x;
}

// The first bin in which a running sum from the top, `upto` (inclusive) at thread `bin`, reaches `need`, and the sum
// before it; BINS if none does.
__device__ __forceinline__ int bin_of(BinScratch& s, uint64_t upto, uint64_t here, uint64_t need, uint64_t& before) {
  __syncthreads();
  if (threadIdx.x == 0) s.bin = BINS, s.before = 0;
  __syncthreads();
  if (threadIdx.x < BINS && upto >= need && upto - here < need) s.bin = threadIdx.x, s.before = upto - here;
  __syncthreads();
  before = s.before;
  return s.bin;
}

// The bin in which min_p cuts, and the step there.
__device__ __forceinline__ int min_p_bin(const Weigher& w, float top, double min_p, int& step) {
  step = INT32_MIN;
  if (!(min_p > 1e-300)) return BINS;
  step = (int)(uint32_t)__builtin_bit_cast(uint64_t, (double)top * w.rate + log2(min_p) + Weigher::magic());
  return (int)min((int64_t)OCTAVE * w.exponent - (step >> 5), (int64_t)BINS);
}

// A workgroup a row (BINS threads, a bin each): joins the parts' bins and finds the first that a filter cuts.
template <class T>
__global__ __launch_bounds__(BINS) void pick_kernel(Args a, Work work) {
  __shared__ BinScratch s;
  __shared__ int apart[MAX_PARTS];
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bin = threadIdx.x;
  const Row<T> r = row_of<T>(a, row);
  const Filters f = filters_of(a, row);
  if (lists_parts(f) || !(r.temperature > 0.)) return;
  const Part mine = part_of(a, work.parts + (int64_t)row * a.parts, lane);
  const RowTop t = row_top(mine);
  if (t.exponent == NOTHING) return;
  RowState state{t.top, t.exponent, BINS, 0, 0, 0, t.exponent == BEYOND || t.exponent < -FAR, 0};
  if (state.search) {
    if (threadIdx.x == 0) work.rows[row] = state;
    return;
  }
  if (wave == 0) apart[lane] = apart_of(t.exponent, mine.exponent);
  __syncthreads();
  const uint64_t* masses = work.masses + (int64_t)row * a.parts * BINS;
  const uint32_t* counts = work.counts + (int64_t)row * a.parts * BINS;
  uint64_t mass = 0, count = 0;
  for (int p0 = 0; p0 < a.parts; p0 += AHEAD) {
    uint64_t m[AHEAD];
    uint32_t n[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {  // (loads first, in flight together)
      const int p = min(p0 + i, a.parts - 1), from = bin - OCTAVE * apart[p];
      const bool there = p0 + i < a.parts && from >= 0 && bin <= OCTAVE * a.shift;
      const int64_t at = there ? (int64_t)p * BINS + from : 0;
      m[i] = there ? masses[at] : 0;
      n[i] = there && a.counting ? counts[at] : 0;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) mass += m[i] >> min(apart[min(p0 + i, a.parts - 1)], 63), count += n[i];
  }
  uint64_t total, ignored, before;
  const uint64_t upto = block_scan<BINS / 64>(s.sums, mass, total);
  work.sums[(int64_t)row * BINS + bin] = upto;
  __shared__ double no_table;
  const Weigher weigher(&no_table, r.temperature, a.shift, t.exponent);
  int cut = BINS;
  if (f.top_k > 0 && f.top_k < a.vocab) {
    const uint64_t count_upto = block_scan<BINS / 64>(s.sums, count, ignored);
    work.count_sums[(int64_t)row * BINS + bin] = (uint32_t)count_upto;
    cut = bin_of(s, count_upto, count, (uint64_t)f.top_k, before);
  }
  if (cut == BINS) {  // (a rank's cut comes first: what top_p is a share of depends on it)
    if (f.top_p < 1.) {
      const uint64_t need = share_of(fmax(f.top_p, 0.), total, true);
      cut = bin_of(s, upto, mass, need ? need : 1, before);
    }
    int step;
    cut = min(cut, min_p_bin(weigher, t.top, f.min_p, step));
  }
  if (threadIdx.x == 0) {
    state.bin = cut;
    if (cut < BINS) {
      state.low = max(weigher.first_key(weigher.bin_step(cut)), order_key(-INFINITY) + 1);
      state.high = weigher.first_key(weigher.bin_step(cut - 1));
    }
    work.rows[row] = state;
  }
}

// Lists the tokens of the bin that is cut, in any order.
template <class T>
__global__ __launch_bounds__(WEIGH_THREADS) void gather_kernel(Args a, Work work) {
  const int part = blockIdx.x, row = blockIdx.y;
  const Row<T> r = row_of<T>(a, row);
  if (lists_parts(filters_of(a, row)) || !(r.temperature > 0.)) return;
  const Part p = work.parts[(int64_t)row * a.parts + part];
  if (p.exponent == NOTHING) return;  // (of a row without any, the state is not set)
  RowState* state = work.rows + row;
  const uint32_t low = state->low, high = state->high;
  if (state->search || state->bin == BINS || order_key(p.top) < low) return;
  __shared__ uint64_t found[LIST];
  __shared__ int n, first;
  if (threadIdx.x == 0) n = 0;
  __syncthreads();
  const int from = part * a.part_len, to = min(a.vocab, from + a.part_len);
  r.template each<16, WEIGH_THREADS>(from + threadIdx.x, to, [&](int i, float x) {
    const uint32_t key = order_key(x);
    if (key >= low && key < high) {
      const int at = atomicAdd(&n, 1);
      if (at < LIST) found[at] = token_of(key, i);
    }
  });
  __syncthreads();
  if (threadIdx.x == 0 && n) first = atomicAdd(&state->listed, n);  // (one of a thousand a row at most: they go one by one)
  __syncthreads();
  for (int i = threadIdx.x; i < n && i < LIST && first + i < LIST; i += WEIGH_THREADS) work.lists[(int64_t)row * LIST + first + i] = found[i];
}

struct DrawScratch {
  union {
    Scratch search;
    struct {
      uint64_t list[LIST];  // tokens of a bin
      uint64_t few[LIST];   // those of them that need ranking: by falling key, then index
    };
  };
  double table[STEPS];
  BinScratch bins;
  uint64_t sub_mass[SUBS];
  uint32_t sub_count[SUBS];
  uint32_t count[BINS];
  uint64_t part_mass[MAX_PARTS];
  int exponents[MAX_PARTS], listed[MAX_PARTS];
  int ranks[THREADS];
  int n, keep, sub;
  uint64_t sub_before;
  uint32_t sub_rank;
};

// few's n values in the order of order(value) (all different): each counts those before it, several threads a value
// where there are few.
template <class Order>
__device__ __forceinline__ void rank_few(DrawScratch& s, int n, Order order) {
  int slices = 1;
  while (slices < 16 && 2 * slices * n <= THREADS) slices *= 2;
  uint64_t x[LIST / THREADS];
  int rank[LIST / THREADS];
  s.ranks[threadIdx.x] = 0;
  __syncthreads();
  if (slices > 1) {
    const int i = threadIdx.x % (THREADS / slices), slice = threadIdx.x / (THREADS / slices);
    if (i < n) {
      const auto mine = order(s.few[i]);
      int before = 0;
#pragma unroll 4
      for (int j = slice; j < n; j += slices) before += order(s.few[j]) < mine;
      atomicAdd(&s.ranks[i], before);
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < LIST / THREADS; ++k) {
    const int i = k * THREADS + threadIdx.x;
    if (i >= n) continue;
    x[k] = s.few[i], rank[k] = slices > 1 ? s.ranks[i] : 0;
    if (slices == 1)
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank[k] += order(s.few[j]) < order(x[k]);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < LIST / THREADS; ++k)
    if (k * THREADS + (int)threadIdx.x < n) s.few[rank[k]] = x[k];
  __syncthreads();
}

// Lists the row's tokens with keys in [low, high) that `cut` takes, reading all of it. Returns how many.
template <class T>
__device__ __forceinline__ int list_tokens(DrawScratch& s, const Row<T>& r, uint32_t low, uint32_t high, const Cut& cut) {
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  r.template each<16, THREADS>(threadIdx.x, r.vocab, [&](int i, float x) {
    const uint32_t key = order_key(x);
    if (key >= low && key < high && cut.takes(key, i)) {
      const int to = atomicAdd(&s.n, 1);
      if (to < LIST) s.list[to] = token_of(key, i);
    }
  });
  __syncthreads();
  return s.n;
}

// How many of few's n ranked tokens stay: at most `most`, up to the one at which the weight, `sum` before them, reaches
// `need`, and while w >= min_p.
template <class T>
__device__ __forceinline__ int kept_of(DrawScratch& s, const Row<T>& r, const Weigher& weigher, int n, int64_t most, uint64_t sum,
                                       uint64_t need, double min_p) {
  __syncthreads();
  if (threadIdx.x == 0) s.keep = (int)min((int64_t)n, most);
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const float x = i < n ? logit_of(key_of(s.few[i])) : -INFINITY;
    uint64_t all;
    const uint64_t upto = sum + block_scan<THREADS / 64>(s.bins.sums, i < n ? weigher.weight(x) : 0, all);
    if (i < n && upto >= need) atomicMin(&s.keep, i + 1);
    if (i < n && min_p > 0. && !(r.weight(x) >= min_p)) atomicMin(&s.keep, i);
    sum += all;
  }
  __syncthreads();
  return s.keep;
}

// Where a filter cuts the bin whose n tokens are listed: after the token at which their weight, `sum` before them,
// reaches `need`, after `rank` of them, or where w < min_p (min_step: the step of that, if it is in this bin). Only the
// tokens of one step are ranked. The cut is never looser than `within`: a step at which min_p cuts may lie below it.
template <class T>
__device__ __forceinline__ Cut cut_bin_at(DrawScratch& s, const Row<T>& r, const Weigher& weigher, int bin, int n, const Cut& within,
                                          uint64_t sum, uint64_t need, int64_t rank, double min_p, int min_step) {
  auto sub_of = [&](uint64_t token) { return SUBS - 1 - (weigher.step(logit_of(key_of(token))) & (SUBS - 1)); };
  auto takes = [&](uint64_t token) { return within.takes(key_of(token), index_of(token)); };
  auto above = [&](uint32_t key) { return key < within.key ? within : Cut{key, -1}; };  // the keys above `key` that `within` takes
  __syncthreads();
  if (threadIdx.x < SUBS) s.sub_mass[threadIdx.x] = 0, s.sub_count[threadIdx.x] = 0;
  if (threadIdx.x == 0) s.n = 0, s.sub = SUBS;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t token = s.list[i];
    if (!takes(token)) continue;
    const int sub = sub_of(token);
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.sub_mass[sub]), (unsigned long long)weigher.weight(logit_of(key_of(token))));
    atomicAdd(&s.sub_count[sub], 1u);
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const uint64_t mass = lane < SUBS ? s.sub_mass[lane] : 0, count = lane < SUBS ? s.sub_count[lane] : 0;
    const uint64_t upto = sum + wave_scan(mass), ranks = wave_scan(count);
    const int min_sub = min_step >> 5 == OCTAVE * weigher.exponent - bin ? SUBS - 1 - (min_step & (SUBS - 1)) : SUBS;
    const uint64_t cuts = __ballot(lane < SUBS && (upto >= need || (int64_t)ranks >= rank || lane == min_sub));
    if (cuts && lane == __ffsll((unsigned long long)cuts) - 1) s.sub = lane, s.sub_before = upto - mass, s.sub_rank = (uint32_t)(ranks - count);
  }
  __syncthreads();
  const int sub = s.sub;
  if (sub == SUBS) return above(weigher.first_key(weigher.bin_step(bin)) - 1);  // (sums a few units short: all of it)
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t token = s.list[i];
    if (takes(token) && sub_of(token) == sub) s.few[atomicAdd(&s.n, 1)] = token;
  }
  __syncthreads();
  const int few = s.n;
  rank_few(s, few, [](uint64_t x) { return x; });
  const int keep = kept_of(s, r, weigher, few, rank - s.sub_rank, s.sub_before, need, min_p);
  if (keep) return Cut{key_of(s.few[keep - 1]), index_of(s.few[keep - 1])};
  return above(few ? key_of(s.few[0]) : weigher.first_key(weigher.bin_step(bin) + SUBS - sub) - 1);
}

// A row whose parts listed what the first top_k can be among: all of it from the lists.
template <class T>
__device__ __forceinline__ bool draw_listed(DrawScratch& s, const Args& a, const Work& work, int row, const Row<T>& r, const Filters& f,
                                            const Weigher& weigher, int64_t* out) {
  // how many tokens the bins down to each hold, then the bin in which that reaches top_k
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t* lists = work.part_list + (int64_t)row * a.parts * PART_LIST;
  for (int i = threadIdx.x; i < BINS; i += THREADS) s.count[i] = 0;
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  auto each = [&](auto g) {  // g(token, bin), a wave a part
    for (int p = wave; p < a.parts; p += THREADS / 64)
      for (int i = lane; i < s.listed[p]; i += 64) {
        const uint64_t token = lists[(int64_t)p * PART_LIST + i];
        int bin;
        if (weigher.weight(logit_of(key_of(token)), bin)) g(token, bin);
      }
  };
  each([&](uint64_t, int bin) { atomicAdd(&s.count[bin], 1u); });
  __syncthreads();
  uint64_t ignored, before;
  const uint64_t here = threadIdx.x < BINS ? s.count[threadIdx.x] : 0;
  const uint64_t upto = block_scan<THREADS / 64>(s.bins.sums, here, ignored);
  const int last = bin_of(s.bins, upto, here, (uint64_t)f.top_k, before);
  each([&](uint64_t token, int bin) {
    if (bin <= last) {
      const int to = atomicAdd(&s.n, 1);
      if (to < LIST) s.few[to] = token;
    }
  });
  __syncthreads();
  int n = s.n;
  if (n > LIST) return false;
  rank_few(s, n, [](uint64_t x) { return x; });
  n = min(n, (int)f.top_k);
  // (top_k is at most SMALL_K: a token a thread from here on)
  uint64_t total;
  const uint64_t w = (int)threadIdx.x < n ? weigher.weight(logit_of(key_of(s.few[threadIdx.x]))) : 0;
  block_scan<THREADS / 64>(s.bins.sums, w, total);
  uint64_t need = ~0ull;
  if (f.top_p < 1.) need = share_of(fmax(f.top_p, 0.), total, true);
  n = kept_of(s, r, weigher, n, n, 0, need ? need : 1, f.min_p);
  // by index, then the token at which the weight passes the target
  rank_few(s, n, [](uint64_t x) { return (uint32_t)x; });
  const uint64_t token = (int)threadIdx.x < n ? s.few[threadIdx.x] : 0;
  const uint64_t weight = (int)threadIdx.x < n ? weigher.weight(logit_of(key_of(token))) : 0;
  const uint64_t sum = block_scan<THREADS / 64>(s.bins.sums, weight, total);
  const uint64_t target = target_of(f.u, total);
  if (target < sum && target >= sum - weight) *out = index_of(token);
  return true;
}

// LISTED: rows whose parts listed their tokens, else the others. (Kernels of their own: in one, with search_row called,
// scalar registers were spilled into vector registers that were spilled themselves, and a value came back wrong.)
template <class T, bool LISTED>
__global__ __launch_bounds__(THREADS) void draw_kernel(Args a, Work work) {
  __shared__ DrawScratch s;
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Row<T> r = row_of<T>(a, row);
  const Filters f = filters_of(a, row);
  if (lists_parts(f) != LISTED) return;
  const Part mine = part_of(a, work.parts + (int64_t)row * a.parts, lane);
  const RowTop t = row_top(mine);
  int64_t* out = a.out + row;
  if (t.exponent == NOTHING || !(r.temperature > 0.)) {
    if (threadIdx.x == 0) *out = t.exponent == NOTHING ? -1 : t.first;
    return;
  }
  r.top = t.top;
  if (t.exponent == BEYOND || t.exponent < -FAR) return search_row(s.search, r, f, out);
  if (wave == 0) s.exponents[lane] = mine.exponent, s.listed[lane] = mine.listed;
  for (int i = threadIdx.x; i < STEPS; i += THREADS) s.table[i] = exp2(i * (1. / STEPS));
  __syncthreads();
  const Weigher weigher(s.table, r.temperature, a.shift, t.exponent);
  if (LISTED) {
    if (__any(mine.listed > PART_LIST) || !draw_listed(s, a, work, row, r, f, weigher, out)) search_row(s.search, r, f, out);
    return;
  }

  const RowState state = work.rows[row];
  const uint64_t* sums = work.sums + (int64_t)row * BINS;
  uint64_t total = sums[BINS - 1];
  const uint64_t upto = threadIdx.x < BINS ? sums[threadIdx.x] : total;
  const uint64_t here = threadIdx.x < BINS ? upto - (threadIdx.x ? sums[threadIdx.x - 1] : 0) : 0;
  Cut cut{order_key(-INFINITY), -1};  // every finite logit
  int cut_bin = state.bin, n = 0;     // the bin that it cuts, whose n tokens are listed: the bins above are whole
  if (cut_bin < BINS) {
    n = state.listed;
    if (n > LIST) return search_row(s.search, r, f, out);
    for (int i = threadIdx.x; i < n; i += THREADS) s.list[i] = work.lists[(int64_t)row * LIST + i];
    const uint32_t* counts = work.count_sums + (int64_t)row * BINS;
    const bool by_rank = f.top_k > 0 && f.top_k < a.vocab && counts[cut_bin] >= (uint64_t)f.top_k;
    if (by_rank) {
      cut = cut_bin_at(s, r, weigher, cut_bin, n, cut, 0, ~0ull, f.top_k - (cut_bin ? (int64_t)counts[cut_bin - 1] : 0), 0., INT32_MIN);
      uint64_t sum = 0, more;
      for (int i = threadIdx.x; i < n; i += THREADS)
        if (cut.takes(key_of(s.list[i]), index_of(s.list[i]))) sum += weigher.weight(logit_of(key_of(s.list[i])));
      block_scan<THREADS / 64>(s.bins.sums, sum, more);
      total = (cut_bin ? sums[cut_bin - 1] : 0) + more;
    }
    uint64_t need = ~0ull, before;
    if (f.top_p < 1.) need = share_of(fmax(f.top_p, 0.), total, true);
    need = need ? need : 1;
    int bin = cut_bin, min_step;
    const int m_bin = min_p_bin(weigher, r.top, f.min_p, min_step);
    if (by_rank) {
      bin = min(m_bin, f.top_p < 1. ? bin_of(s.bins, upto, here, need, before) : BINS);
      if (bin < cut_bin) {  // another bin is cut: its tokens are to be found first
        n = list_tokens(s, r, weigher.first_key(weigher.bin_step(bin)), weigher.first_key(weigher.bin_step(bin - 1)), cut);
        if (n > LIST) return search_row(s.search, r, f, out);
        cut_bin = bin;
      }
    }
    if (bin <= cut_bin) cut = cut_bin_at(s, r, weigher, bin, n, cut, bin ? sums[bin - 1] : 0, need, INT64_MAX, f.min_p, min_step);
  }

  // the kept weight of every part: whole bins, and what the cut one keeps
  const uint64_t* masses = work.masses + (int64_t)row * a.parts * BINS;
  if (threadIdx.x < MAX_PARTS) s.part_mass[threadIdx.x] = 0;
  __syncthreads();
  for (int p = wave; p < a.parts; p += THREADS / 64) {
    const int apart = apart_of(t.exponent, s.exponents[p]), end = min(cut_bin, OCTAVE * a.shift + 1) - OCTAVE * apart;
    uint64_t m[BINS / 64], sum = 0;
#pragma unroll
    for (int i = 0; i < BINS / 64; ++i) m[i] = 64 * i + lane < end ? masses[(int64_t)p * BINS + 64 * i + lane] : 0;
#pragma unroll
    for (int i = 0; i < BINS / 64; ++i) sum += m[i] >> min(apart, 63);
    sum = wave_scan(sum);
    if (lane == 63) s.part_mass[p] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t token = s.list[i];
    if (cut.takes(key_of(token), index_of(token)))
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.part_mass[index_of(token) / a.part_len]),
                (unsigned long long)weigher.weight(logit_of(key_of(token))));
  }
  __syncthreads();
  const uint64_t parts_upto = wave_scan(s.part_mass[lane]);  // lane p: the kept weight of parts up to p
  total = shfl64(parts_upto, 63);
  uint64_t target = target_of(f.u, total);
  const int part = __ffsll((unsigned long long)__ballot(parts_upto > target)) - 1;
  target -= shfl64(parts_upto, part) - s.part_mass[part];

  // The part, in order: a consecutive run of tokens a thread. Weights in the part's own unit, in which its bins hold their
  // sums: tokens lighter than the row's unit, a few of which can make the part's mass, are none there.
  const int from = part * a.part_len, to = min(a.vocab, from + a.part_len), run = (to - from + THREADS - 1) / THREADS;
  const int begin = min(to, from + (int)threadIdx.x * run), end = min(to, begin + run);
  const int apart = apart_of(t.exponent, s.exponents[part]);  // (at most `shift`, as the part has mass)
  const Weigher inside(s.table, r.temperature, a.shift, s.exponents[part]);
  auto kept = [&](int i, float x) -> uint64_t {
    if (!cut.takes(order_key(x), i)) return 0;
    int bin;
    const uint64_t w = inside.weight(x, bin);
    return bin + OCTAVE * apart <= OCTAVE * a.shift ? w : 0;  // (of the row's bins, as the part's mass)
  };
  uint64_t sum = 0, all;
  r.template each<8, 1>(begin, end, [&](int i, float x) { sum += kept(i, x); });
  uint64_t passed = block_scan<THREADS / 64>(s.bins.sums, sum, all);
  // The part's mass is each bin's sum rounded down to the row's unit, so `all` is that many units or a few more: they go
  // to the last one.
  target = target + 1 == s.part_mass[part] ? all - 1 : target << apart;
  if (target >= passed || target < passed - sum) return;
  passed -= sum;
  int token = -1;
  r.template each<8, 1>(begin, end, [&](int i, float x) {
    passed += kept(i, x);
    if (token < 0 && passed > target) token = i;
  });
  *out = token;
}

static int parts_of(int rows, int vocab) {
  // parts of 2048 tokens and more, while two thousand workgroups find work
  const int64_t most = (vocab + 2047) / 2048, want = (2048 + rows - 1) / rows;
  const int64_t n = most < want ? most : want;
  return n < MAX_PARTS ? (int)n : MAX_PARTS;
}

// Workspace of `rows` rows (at most ROWS at a time), laid out at `at`; returns its bytes.
static int64_t work_of(int rows, int vocab, void* at, Work* w) {
  const int64_t n = rows < ROWS ? rows : ROWS, slots = n * parts_of((int)n, vocab);
  uint8_t* p = static_cast<uint8_t*>(at);
  int64_t bytes = 0;
  auto take = [&](int64_t size) {
    const int64_t here = bytes;
    bytes += (size + 255) & ~(int64_t)255;
    return p + here;
  };
  Work x;
  x.masses = reinterpret_cast<uint64_t*>(take(slots * BINS * 8));
  x.part_list = reinterpret_cast<uint64_t*>(take(slots * PART_LIST * 8));
  x.sums = reinterpret_cast<uint64_t*>(take(n * BINS * 8));
  x.lists = reinterpret_cast<uint64_t*>(take(n * LIST * 8));
  x.parts = reinterpret_cast<Part*>(take(slots * (int64_t)sizeof(Part)));
  x.rows = reinterpret_cast<RowState*>(take(n * (int64_t)sizeof(RowState)));
  x.counts = reinterpret_cast<uint32_t*>(take(slots * BINS * 4));
  x.count_sums = reinterpret_cast<uint32_t*>(take(n * BINS * 4));
  if (w) *w = x;
  return bytes;
}

template <class T>
static void launch(const Args& a, int rows, const Work& work, bool some_listed, bool all_listed, hipStream_t st) {
  hipLaunchKernelGGL(weigh_kernel<T>, dim3(a.parts, rows), dim3(WEIGH_THREADS), 0, st, a, work);
  if (!all_listed) {
    hipLaunchKernelGGL(pick_kernel<T>, dim3(rows), dim3(BINS), 0, st, a, work);
    hipLaunchKernelGGL(gather_kernel<T>, dim3(a.parts, rows), dim3(WEIGH_THREADS), 0, st, a, work);
    hipLaunchKernelGGL((draw_kernel<T, false>), dim3(rows), dim3(THREADS), 0, st, a, work);
  }
  if (some_listed) hipLaunchKernelGGL((draw_kernel<T, true>), dim3(rows), dim3(THREADS), 0, st, a, work);
}

}  // namespace sample
}  // namespace dkv

using namespace dkv;

extern "C" {

int64_t dkv_sample_workspace_bytes(int32_t rows, int32_t vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > 1 << 22) return 0;
  return sample::work_of(rows, vocab, nullptr, nullptr);
}

int dkv_sample(const void* logits, int32_t dtype, int64_t row_stride, int32_t rows, int32_t vocab, const void* u, int32_t u_dtype,
               const dkv_sampling* sampling, int64_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
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
  const int64_t need = dkv_sample_workspace_bytes(rows, vocab);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need) {
    set_error("dkv_sample: workspace of %lld bytes needed, %lld given (16-byte aligned)", (long long)need, (long long)workspace_bytes);
    return DKV_EINVAL;
  }
  sample::Args a{};
  a.logits = logits, a.u = u, a.row_stride = row_stride, a.out = out;
  a.vocab = vocab, a.u_dtype = u_dtype, a.p = p;
  a.shift = 62;
  while (a.shift > 50 || ((uint64_t)vocab >> (62 - a.shift)) > 0) --a.shift;  // vocab << shift stays below 2^62
  a.parts = sample::parts_of(rows < sample::ROWS ? rows : sample::ROWS, vocab);
  a.part_len = (vocab + a.parts - 1) / a.parts;
  a.counting = p.top_k_rows || (p.top_k > 0 && p.top_k < vocab);
  sample::Work work;
  sample::work_of(rows, vocab, workspace, &work);
  const bool all_listed = !p.top_k_rows && p.top_k > 0 && p.top_k <= sample::SMALL_K;
  for (int at = 0; at < rows; at += sample::ROWS) {
    const int n = rows - at < sample::ROWS ? rows - at : sample::ROWS;
    sample::Args b = a;
    b.logits = static_cast<const uint8_t*>(logits) + at * row_stride * (dtype == 0 ? 2 : 4);
    b.u = static_cast<const uint8_t*>(u) + (int64_t)at * (u_dtype ? 8 : 4);
    b.out = out + at;
    if (p.temperature_rows) b.p.temperature_rows += at;
    if (p.top_p_rows) b.p.top_p_rows += at;
    if (p.min_p_rows) b.p.min_p_rows += at;
    if (p.top_k_rows) b.p.top_k_rows += at;
    if (dtype == 0) sample::launch<uint16_t>(b, n, work, p.top_k_rows || all_listed, all_listed, (hipStream_t)stream);
    else sample::launch<float>(b, n, work, p.top_k_rows || all_listed, all_listed, (hipStream_t)stream);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
