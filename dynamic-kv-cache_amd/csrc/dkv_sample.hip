// Sampling (gfx950): one token a row from logits and a given random number.
//
// w_i = exp((x_i - max) / temperature); of the tokens in order of their logits (equal ones: the first) the first
// top_k, of those the shortest run that holds top_p of their weight, of those the ones with w >= min_p; then the
// first token, in the vocabulary's order, up to which the kept weight exceeds u times its total.
//
// Two launches. weigh_kernel: many workgroups a row sum the weights of their part of the vocabulary by bins, eight an
// octave, so that a bin's tokens are consecutive in the order of the logits. draw_kernel, a workgroup a row: finds the
// bins in which the filters cut, lists and ranks the few tokens of those bins, then finds the part and the token where
// the kept weight passes the target. Weights are computed in 64 bits and summed as integers (multiples of 2^-SHIFT of
// a power of two above the largest): such sums are exact and the same in every order, so neither atomics nor the split
// into parts can move a border between two tokens. SHIFT leaves room for a whole vocabulary's sum (40 for 4 million
// tokens, 46 for 49280), and what is lighter counts as nothing.
// What does not fit that (an infinite logit, exponents beyond 65536, more than LIST tokens in a bin that is cut)
// takes search_row, a radix search over the whole row, in the same launch.
#include "dkv_select.h"

namespace dkv {
namespace sample {

constexpr int THREADS = 1024;

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
__device__ __noinline__ void search_row(Scratch& s, const Row<T>& r, const Filters& f, int64_t* out) {
  const int vocab = r.vocab;
  const int64_t top_k = f.top_k;
  const double top_p = f.top_p, min_p = f.min_p;
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
constexpr int OCTAVE = 8, BINS = 512;  // bins of an octave of weight; 52 octaves and more
constexpr int STEPS = 256;             // steps of the table of 2^f
constexpr int LIST = 4096;             // tokens of a bin that is cut
constexpr int MAX_PARTS = 64;
constexpr int AHEAD = 8;  // parts whose bins a thread has in flight
constexpr int NOTHING = INT32_MIN, BEYOND = INT32_MAX;
constexpr double FAR = 65536.;         // largest exponent whose weights keep 2^-36 of their value

struct Part {
  uint32_t key;   // its largest logit, and the first index of it
  int first;
  int exponent;   // its weights are below 2^exponent: the unit of its sums is 2^(exponent - SHIFT)
  int pad;
};

// A logit's base-2 exponent Y = x log2(e) / T as octave + f, and 2^f in [1, 2) as 53 bits: a table of 2^(j / 256) and
// the exponential's series for the rest (below ln 2 / 256, so its fifth term is below 2^-49).
struct Weigher {
  const double* table;
  double rate;  // log2(e) / T
  int shift;
  __device__ __forceinline__ double exponent(float x) const { return (double)x * rate; }
  // Bin from the top of `exponent` down, 8 an octave, and the weight in units of 2^(exponent - shift), rounded down;
  // weight 0 where that is nothing. x is finite.
  __device__ __forceinline__ uint64_t weight(float x, int exponent_, int& bin) const {
    const double y = exponent(x), octave = floor(y), f = y - octave;
    const double down = (double)exponent_ - octave;  // at least 1
    bin = BINS;
    if (!(down <= (double)shift)) return 0;
    const int j = min((int)(f * STEPS), STEPS - 1);
    const double t = (f - j * (1. / STEPS)) * 0.69314718055994530942;
    double e = __builtin_fma(t, 1. / 24, 1. / 6);
    e = __builtin_fma(t, e, .5);
    e = __builtin_fma(t, e, 1.);
    const double w = __builtin_fma(t * table[j], e, table[j]);
    const int d = (int)down;
    bin = OCTAVE * d - 1 - j / (STEPS / OCTAVE);
    const uint64_t bits = __builtin_bit_cast(uint64_t, w);
    // (a series that rounds up to 2 keeps its octave's last value)
    const uint64_t mantissa = bits >= 0x4000000000000000ull ? (1ull << 53) - 1 : (bits & ((1ull << 52) - 1)) | 1ull << 52;
    return mantissa >> (52 - shift + d);
  }
};

template <class T>
__global__ __launch_bounds__(WEIGH_THREADS) void weigh_kernel(Args a, Part* parts, uint64_t* masses, uint32_t* counts) {
  __shared__ double table[STEPS];
  __shared__ uint64_t mass[BINS];
  __shared__ uint32_t count[BINS];
  __shared__ uint32_t best[WEIGH_THREADS / 64];
  __shared__ int at[WEIGH_THREADS / 64];
  const int part = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Row<T> r = row_of<T>(a, row);
  const int from = part * a.part_len, to = min(a.vocab, from + a.part_len);
  for (int i = threadIdx.x; i < STEPS; i += WEIGH_THREADS) table[i] = exp2(i * (1. / STEPS));
  for (int i = threadIdx.x; i < BINS; i += WEIGH_THREADS) mass[i] = 0, count[i] = 0;
  uint32_t top = 0;
  int first = to;
  r.template each<8, WEIGH_THREADS>(from + threadIdx.x, to, [&](int i, float x) {
    const uint32_t key = order_key(x);
    if (key > top) top = key, first = i;
  });
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)top, d, 64);
    const int oi = __shfl_xor(first, d, 64);
    if (o > top || (o == top && oi < first)) top = o, first = oi;
  }
  if (lane == 0) best[wave] = top, at[wave] = first;
  __syncthreads();
  top = best[0], first = at[0];
#pragma unroll
  for (int w = 1; w < WEIGH_THREADS / 64; ++w)
    if (best[w] > top || (best[w] == top && at[w] < first)) top = best[w], first = at[w];
  const Weigher weigher{table, r.temperature > 0. ? 1.44269504088896340736 / r.temperature : 0., a.shift};
  const float x_top = logit_of(top);
  const double y_top = weigher.exponent(x_top);
  const int64_t slot = (int64_t)row * a.parts + part;
  int exponent = NOTHING;
  if (top > order_key(-INFINITY))  // (a part far below the others, of masked tokens say, just adds nothing)
    exponent = x_top < INFINITY && y_top <= FAR ? (int)fmax(floor(y_top) + 1., -1e9) : BEYOND;
  if (threadIdx.x == 0) parts[slot] = Part{top, first, exponent, 0};
  if (!(r.temperature > 0.)) return;
  if (exponent != NOTHING && exponent != BEYOND) {
    r.template each<8, WEIGH_THREADS>(from + threadIdx.x, to, [&](int, float x) {
      if (!(x > -INFINITY)) return;
      int bin;
      const uint64_t w = weigher.weight(x, exponent, bin);
      if (w) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&mass[bin]), (unsigned long long)w);
        if (a.counting) atomicAdd(&count[bin], 1u);
      }
    });
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += WEIGH_THREADS) {
    masses[slot * BINS + i] = mass[i];
    if (a.counting) counts[slot * BINS + i] = count[i];
  }
}

struct DrawScratch {
  union {
    Scratch search;
    struct {
      uint64_t list[LIST];    // ~key << 32 | index, as found
      uint64_t ranked[LIST];  // the same by falling key, then index
    };
  };
  double table[STEPS];
  uint64_t mass[BINS];  // of all parts, and sums from the top
  uint32_t count[BINS];
  uint64_t half_mass[BINS];
  uint32_t half_count[BINS];
  uint64_t sums[THREADS / 64];
  uint64_t part_mass[MAX_PARTS];
  int exponents[MAX_PARTS];
  int listed, bin;
  uint64_t before;
};

// The first bin up to which `sums` (running, from the top) reaches `need`, and the sum before it; BINS if none does.
template <class T>
__device__ __forceinline__ int bin_of(DrawScratch& s, const T* sums, uint64_t need, uint64_t& before) {
  __syncthreads();
  if (threadIdx.x == 0) s.bin = BINS;
  __syncthreads();
  if (threadIdx.x < BINS) {
    const uint64_t here = sums[threadIdx.x], above = threadIdx.x ? (uint64_t)sums[threadIdx.x - 1] : 0;
    if (here >= need && above < need) s.bin = threadIdx.x, s.before = above;
  }
  __syncthreads();
  before = s.before;
  return s.bin;
}

__device__ __forceinline__ uint64_t block_scan(DrawScratch& s, uint64_t x, uint64_t& total) {  // inclusive
  x = wave_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.sums[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += s.sums[w];
    total += s.sums[w];
  }
  return before + x;
}

// The smallest logit's key whose exponent is at least `floor8` eighths (the same arithmetic as weight()'s bin).
__device__ __forceinline__ uint32_t first_key(const Weigher& w, double floor8) {
  float x = (float)(floor8 / (8. * w.rate));
  x = fminf(fmaxf(x, -3.4028235e38f), 3.4028235e38f);
  uint32_t key = order_key(x);
  for (int i = 0; i < 8 && floor(8. * w.exponent(logit_of(key - 1))) >= floor8; ++i) --key;
  for (int i = 0; i < 8 && floor(8. * w.exponent(logit_of(key))) < floor8; ++i) ++key;
  return key;
}

// Lists the row's tokens with keys in [low, high) that `cut` takes, ranked by falling key, then index. Returns how
// many, or more than LIST if they do not fit.
template <class T>
__device__ __forceinline__ int rank_tokens(DrawScratch& s, const Row<T>& r, uint32_t low, uint32_t high, const Cut& cut) {
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  r.template each<16, THREADS>(threadIdx.x, r.vocab, [&](int i, float x) {
    const uint32_t key = order_key(x);
    if (key >= low && key < high && cut.takes(key, i)) {
      const int to = atomicAdd(&s.listed, 1);
      if (to < LIST) s.list[to] = (uint64_t)~key << 32 | (uint32_t)i;
    }
  });
  __syncthreads();
  const int n = s.listed;
  if (n > LIST) return n;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t x = s.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.list[j] < x;
    s.ranked[rank] = x;
  }
  __syncthreads();
  return n;
}

__device__ __forceinline__ uint32_t key_at(const DrawScratch& s, int i) { return ~(uint32_t)(s.ranked[i] >> 32); }

template <class T>
__global__ __launch_bounds__(THREADS) void draw_kernel(Args a, const Part* parts, const uint64_t* masses, const uint32_t* counts) {
  __shared__ DrawScratch s;
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Row<T> r = row_of<T>(a, row);
  const Filters f = filters_of(a, row);
  parts += (int64_t)row * a.parts, masses += (int64_t)row * a.parts * BINS, counts += (int64_t)row * a.parts * BINS;
  Part best = lane < a.parts ? parts[lane] : Part{0, 0, NOTHING, 0};  // lane p has part p (MAX_PARTS is a wave)
  if (wave == 0) s.exponents[lane] = best.exponent;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t key = (uint32_t)__shfl_xor((int)best.key, d, 64);
    const int at = __shfl_xor(best.first, d, 64), e = __shfl_xor(best.exponent, d, 64);
    if (key > best.key || (key == best.key && at < best.first)) best.key = key, best.first = at;
    best.exponent = max(best.exponent, e);
  }
  const uint32_t top = best.key;
  const int first = best.first, exponent = best.exponent;
  int64_t* out = a.out + row;
  if (exponent == NOTHING || !(r.temperature > 0.)) {
    if (threadIdx.x == 0) *out = exponent == NOTHING ? -1 : first;
    return;
  }
  r.top = logit_of(top);
  if (exponent == BEYOND || exponent < -FAR) return search_row(s.search, r, f, out);
  const Weigher weigher{s.table, 1.44269504088896340736 / r.temperature, a.shift};
  for (int i = threadIdx.x; i < STEPS; i += THREADS) s.table[i] = exp2(i * (1. / STEPS));
  __syncthreads();

  // octaves from the row's exponent down to a part's (more than any weight has where the part has none)
  auto apart_of = [&](int p) { return s.exponents[p] == NOTHING ? BINS : (int)min((int64_t)exponent - s.exponents[p], (int64_t)BINS); };
  // the row's bins, running sums from the top
  uint64_t mine = 0;
  uint32_t mine_count = 0;
  const int bins = OCTAVE * a.shift;  // in those below a token weighs nothing
  for (int p = wave / (BINS / 64); p < MAX_PARTS; p += 2 * AHEAD) {  // half of the threads take the odd parts
    if (p >= a.parts) break;
    uint64_t m[AHEAD];
    uint32_t n[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {  // (loads first, in flight together)
      const int part = p + 2 * i, bin = threadIdx.x % BINS - OCTAVE * min(apart_of(min(part, a.parts - 1)), BINS);
      const bool there = part < a.parts && bin >= 0 && threadIdx.x % BINS < bins;
      const int64_t at = there ? (int64_t)part * BINS + bin : 0;
      m[i] = masses[at] & (there ? ~0ull : 0ull);
      n[i] = a.counting && there ? counts[at] : 0u;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      mine += m[i] >> min(apart_of(min(p + 2 * i, a.parts - 1)), 63), mine_count += n[i];
  }
  if (threadIdx.x >= BINS) s.half_mass[threadIdx.x % BINS] = mine, s.half_count[threadIdx.x % BINS] = mine_count;
  __syncthreads();
  if (threadIdx.x < BINS) mine += s.half_mass[threadIdx.x], mine_count += s.half_count[threadIdx.x];
  else mine = mine_count = 0;
  uint64_t total, ignored;
  mine = block_scan(s, mine, total);
  if (threadIdx.x < BINS) s.mass[threadIdx.x] = mine;
  if (a.counting) {
    mine = block_scan(s, mine_count, ignored);
    if (threadIdx.x < BINS) s.count[threadIdx.x] = (uint32_t)mine;
  }
  // the keys of a bin: [low, high)
  auto bin_keys = [&](int bin, uint32_t& low, uint32_t& high) {
    const double floor8 = (double)OCTAVE * exponent - 1 - bin;
    low = first_key(weigher, floor8), high = first_key(weigher, floor8 + 1);
  };
  auto weight = [&](uint32_t key) {
    int bin;
    return weigher.weight(logit_of(key), exponent, bin);
  };

  Cut cut{order_key(-INFINITY), -1};  // every finite logit
  int cut_bin = BINS;                 // the bin that it cuts: those above are whole
  int listed = 0;                     // tokens of that bin, ranked
  if (f.top_k > 0 && f.top_k < a.vocab) {
    uint64_t before;
    const int bin = bin_of(s, s.count, (uint64_t)f.top_k, before);
    if (bin < BINS) {
      uint32_t low, high;
      bin_keys(bin, low, high);
      const int n = rank_tokens(s, r, low, high, cut), keep = (int)(f.top_k - (int64_t)before);
      if (n > LIST) return search_row(s.search, r, f, out);
      total = bin ? s.mass[bin - 1] : 0;
      uint64_t sum = 0;
      for (int i = threadIdx.x; i < keep && i < n; i += THREADS) sum += weight(key_at(s, i));
      uint64_t more;
      block_scan(s, sum, more);
      total += more;
      const int last = min(keep, n) - 1;
      cut = Cut{key_at(s, last), (int)(uint32_t)s.ranked[last]}, cut_bin = bin, listed = n;
    }
  }
  if (f.top_p < 1. || f.min_p > 0.) {
    uint64_t need = ~0ull, before = 0;
    int p_bin = BINS, m_bin = BINS;
    if (f.top_p < 1.) {
      need = share_of(fmax(f.top_p, 0.), total, true);
      need = need ? need : 1;
      p_bin = bin_of(s, s.mass, need, before);
    }
    if (f.min_p > 0.) {
      const double at = (double)OCTAVE * exponent - 1 - floor(8. * (weigher.exponent(r.top) + log2(f.min_p)));
      m_bin = at < BINS ? (int)at : BINS;
    }
    const int bin = min(p_bin, m_bin);
    if (bin < BINS && bin <= cut_bin) {
      uint32_t low, high;
      bin_keys(bin, low, high);
      const int n = rank_tokens(s, r, low, high, cut);
      if (n > LIST) return search_row(s.search, r, f, out);
      // the first `keep` of the ranked tokens stay
      __syncthreads();
      if (threadIdx.x == 0) s.listed = n;
      __syncthreads();
      uint64_t sum = bin ? s.mass[bin - 1] : 0;
      for (int i0 = 0; i0 < n; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < n ? key_at(s, i) : 0u;
        uint64_t here = i < n ? weight(key) : 0, all;
        const uint64_t upto = sum + block_scan(s, here, all);
        if (i < n && bin == p_bin && upto >= need) atomicMin(&s.listed, i + 1);
        if (i < n && bin == m_bin && !(r.weight(logit_of(key)) >= f.min_p)) atomicMin(&s.listed, i);
        sum += all;
      }
      __syncthreads();
      const int keep = s.listed;
      cut = keep ? Cut{key_at(s, keep - 1), (int)(uint32_t)s.ranked[keep - 1]} : Cut{high - 1, -1};
      cut_bin = bin, listed = n;
    }
  }

  // the kept weight of every part: whole bins, and what the cut one keeps (its tokens are listed)
  if (threadIdx.x < MAX_PARTS) s.part_mass[threadIdx.x] = 0;
  __syncthreads();
  for (int p = wave; p < a.parts; p += THREADS / 64) {
    const int apart = apart_of(p);
    if (apart > a.shift) continue;
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < BINS / 64; ++i)
      if (const int b = 64 * i + lane; b < min(cut_bin, bins) - apart * OCTAVE) sum += masses[(int64_t)p * BINS + b] >> apart;
    sum = wave_scan(sum);
    if (lane == 63) s.part_mass[p] = sum;
  }
  __syncthreads();
  if (cut_bin < BINS)
    for (int i = threadIdx.x; i < listed; i += THREADS) {
      const uint32_t key = key_at(s, i);
      const int token = (int)(uint32_t)s.ranked[i];
      if (cut.takes(key, token))
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.part_mass[token / a.part_len]), (unsigned long long)weight(key));
    }
  __syncthreads();
  const uint64_t parts_upto = wave_scan(s.part_mass[lane]);  // lane p: the kept weight of parts up to p
  total = shfl64(parts_upto, 63);
  uint64_t target = target_of(f.u, total);
  const int part = __ffsll((unsigned long long)__ballot(parts_upto > target)) - 1;
  target -= shfl64(parts_upto, part) - s.part_mass[part];

  // the part, in order: a consecutive run of tokens a thread
  const int from = part * a.part_len, to = min(a.vocab, from + a.part_len), run = (to - from + THREADS - 1) / THREADS;
  const int begin = min(to, from + (int)threadIdx.x * run), end = min(to, begin + run);
  auto kept = [&](int i) -> uint64_t {
    const uint32_t key = order_key(r.at(i));
    return cut.takes(key, i) ? weight(key) : 0;
  };
  uint64_t sum = 0, all;
  for (int i = begin; i < end; ++i) sum += kept(i);
  uint64_t upto = block_scan(s, sum, all);
  // (bins' sums were rounded down once, tokens' one by one: their total may be a few units short)
  if (target >= all) target = all - 1;
  if (all == 0 || target >= upto || target < upto - sum) return;
  upto -= sum;
  for (int i = begin; i < end; ++i) {
    upto += kept(i);
    if (upto > target) {
      *out = i;
      return;
    }
  }
}

static int parts_of(int rows, int vocab) {
  // parts of 2048 tokens and more, while two thousand workgroups find work
  const int64_t most = (vocab + 2047) / 2048, want = (2048 + rows - 1) / rows;
  const int64_t n = most < want ? most : want;
  return n < MAX_PARTS ? (int)n : MAX_PARTS;
}

template <class T>
static void launch(const Args& a, int rows, Part* parts, uint64_t* masses, uint32_t* counts, hipStream_t st) {
  hipLaunchKernelGGL(weigh_kernel<T>, dim3(a.parts, rows), dim3(WEIGH_THREADS), 0, st, a, parts, masses, counts);
  hipLaunchKernelGGL(draw_kernel<T>, dim3(rows), dim3(THREADS), 0, st, a, parts, masses, counts);
}

}  // namespace sample
}  // namespace dkv

using namespace dkv;

extern "C" {

int64_t dkv_sample_workspace_bytes(int32_t rows, int32_t vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > 1 << 22) return 0;
  return (int64_t)rows * sample::parts_of(rows, vocab) * (sizeof(sample::Part) + sample::BINS * (8 + 4));
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
  a.parts = sample::parts_of(rows, vocab), a.part_len = (vocab + a.parts - 1) / a.parts;
  a.counting = p.top_k_rows || (p.top_k > 0 && p.top_k < vocab);
  const int64_t slots = (int64_t)rows * a.parts;
  uint64_t* masses = static_cast<uint64_t*>(workspace);
  sample::Part* parts = reinterpret_cast<sample::Part*>(masses + slots * sample::BINS);
  uint32_t* counts = reinterpret_cast<uint32_t*>(parts + slots);
  const hipStream_t st = (hipStream_t)stream;
  // (the second grid dimension holds 65535 rows)
  for (int at = 0; at < rows; at += 65535) {
    const int n = rows - at < 65535 ? rows - at : 65535;
    sample::Args b = a;
    b.logits = static_cast<const uint8_t*>(logits) + at * row_stride * (dtype == 0 ? 2 : 4);
    b.u = static_cast<const uint8_t*>(u) + (int64_t)at * (u_dtype ? 8 : 4);
    b.out = out + at;
    if (p.temperature_rows) b.p.temperature_rows += at;
    if (p.top_p_rows) b.p.top_p_rows += at;
    if (p.min_p_rows) b.p.min_p_rows += at;
    if (p.top_k_rows) b.p.top_k_rows += at;
    const int64_t slot = (int64_t)at * a.parts;
    if (dtype == 0) sample::launch<uint16_t>(b, n, parts + slot, masses + slot * sample::BINS, counts + slot * sample::BINS, st);
    else sample::launch<float>(b, n, parts + slot, masses + slot * sample::BINS, counts + slot * sample::BINS, st);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
