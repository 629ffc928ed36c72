// Attention over pages, sequences (and groups that share pages) of few query rows (gfx950).
//
// o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = q k_j / 8, over the history's rows and the new ones up to a query's own, in
// one pass with a running maximum m. A workgroup takes 16 query rows (tokens times query heads) of a KV head over a range of units
// of 64 keys, each of its four waves a fourth of these; a step's ranges are cut so that about 2048 workgroups share its units
// whatever the lengths (dkv_paged.hip), and partial rows are joined by merge_kernel. Per half page and wave: keys straight from
// global memory into the operands of S^T = K Q^T (16x16x32 bf16), whose result lies where O^T = V^T P^T reads P^T, values into V^T's.
// No LDS but for scales and the waves' join.
// Weights: sums and statistics in 32 bits; P is the sum of two bf16 values (2^-16) at precision and output bf16, of three (2^-24) at
// fp32 of either. At precision bf16 a packed value is rounded to bf16, GPUCache's rounding; at fp32 its code is multiplied and its scale and offset
// come apart.
// What bounds it: long histories their bytes, six of 30k to 131k tokens of 8 heads at fp32 506 MB in 100 us (5.0 TB/s, of a large
// copy's 5.2), a token of each of 64 streams of 300 to 8128 tokens 107 MB in 27 us; short ones the chain of loads of one launch
// (three of up to 333 tokens 7.5 us); branches the unpacking of shared pages once for each 16 of their rows (48 of 8128 shared
// tokens 15.8 us).
#pragma once
#include "dkv_rows.h"
#include "dkv_paged.h"

namespace dkv {
namespace paged {
namespace few {

using namespace rows;

constexpr int HALF = 32;  // keys at a time

// Half a unit's rows: a page's, or new tokens', from `k` and `v` on. Rows [0, rows) are there.
struct Half {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* scales;        // a packed page's: lane l's (offset, scale) pair, of key l or value l - 32
  uint32_t k_stride, v_stride;  // of new tokens: bytes from row to row, below 2^24
  int rows;
};

// What a lane has loaded: of keys 16 b + c the elements [16 g, 16 g + 16), of values 16 b + 4 g + i the elements
// [4 c, 4 c + 4), and one (offset, scale) pair, which goes to the lanes that need it through LDS (each lane's own copies
// of them would be 20 to 32 registers).
template <int BITS>
struct Loaded {
  uint32_t k[2][BITS / 2], v[2][4][BITS == 16 ? 2 : 1];
  float2 pair;
};

// Rows that a half page does not hold are read too (what is there meets no score and no weight): without a test a lane's
// rows are one address and constant distances. Of new tokens (NEW) the row past the last one is its first again.
template <int BITS, bool NEW = false>
__device__ __forceinline__ void load_keys(const Half& u, int c, int g, Loaded<BITS>& x) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int row = 16 * b + c;
    const uint8_t* at = NEW ? u.k + (__umul24(row < u.rows ? row : 0, u.k_stride) + g * 2 * BITS)
                            : u.k + (uint32_t)(c * 8 * BITS + g * 2 * BITS) + 16 * b * 8 * BITS;
    if (BITS == 4) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(at);
      x.k[b][0] = w[0], x.k[b][1] = w[1];
    } else {
#pragma unroll
      for (int i = 0; i < BITS / 8; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(at + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) x.k[b][4 * i + j] = w[j];
      }
    }
  }
  if (BITS < 16) x.pair = *reinterpret_cast<const float2*>(u.scales);
}

template <int BITS, bool NEW = false>
__device__ __forceinline__ void load_vals(const Half& u, int c, int g, Loaded<BITS>& x) {
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * b + 4 * g + i;
      const uint8_t* at = NEW ? u.v + (__umul24(row < u.rows ? row : 0, u.v_stride) + c * BITS / 2)
                              : u.v + (uint32_t)(4 * g * 8 * BITS + c * BITS / 2) + (16 * b + i) * 8 * BITS;
      if (BITS == 4) {
        x.v[b][i][0] = *reinterpret_cast<const uint16_t*>(at);
      } else if (BITS == 8) {
        x.v[b][i][0] = *reinterpret_cast<const uint32_t*>(at);
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
        x.v[b][i][0] = w[0], x.v[b][i][1 % (BITS == 16 ? 2 : 1)] = w[1];
      }
    }
}

// Codes e and e + 1 of packed words as a bf16 pair: their values (c * scale + offset, each step rounded) at PREC 0, else the
// codes less CENTRE, which bf16 holds exactly; scale and offset come later. (Sums of codes that are not centred cancel
// against their offsets': relative errors of 2.6e-6 in place of 1.1e-6 over 131k tokens.) Nibbles are bytes of two words first, centred codes
// signed bytes, so that a code is one conversion.
template <int BITS, int PREC>
struct Codes {
  uint32_t w[BITS == 4 ? 2 : 1];
};
template <int BITS, int PREC>
__device__ __forceinline__ Codes<BITS, PREC> codes_of(uint32_t w) {
  Codes<BITS, PREC> x;
  if (BITS == 4) x.w[0] = w & 0x0f0f0f0fu, x.w[BITS == 4 ? 1 : 0] = (w >> 4) & 0x0f0f0f0fu;
  else x.w[0] = w;
  if (PREC)
#pragma unroll
    for (int i = 0; i < (BITS == 4 ? 2 : 1); ++i) x.w[i] = (BITS == 4 ? x.w[i] + 0x78787878u : x.w[i]) ^ 0x80808080u;
  return x;
}
template <int BITS, int PREC>
__device__ __forceinline__ float code(const Codes<BITS, PREC>& x, int e) {
  const uint32_t w = x.w[BITS == 4 ? e % 2 : 0] >> (8 * (BITS == 4 ? e / 2 : e));
  return PREC ? (float)(int8_t)w : (float)(w & 255u);
}
template <int PREC>
__device__ __forceinline__ uint32_t values(float c0, float c1, float scale0, float offset0, float scale1, float offset1) {
  return PREC ? pack_bf16(c0, c1) : pack_bf16(c0 * scale0 + offset0, c1 * scale1 + offset1);
}

// A wave's 32 pairs of keys, then of values, to be read by any of its lanes (at PREC 1 with the offset of centred codes).
template <int BITS, int PREC>
__device__ __forceinline__ void share_scales(float2* lds, int lane, float2 mine, int rows) {
  if (PREC) mine.x = __builtin_fmaf(mine.y, CENTRE<BITS == 16 ? 8 : BITS>, mine.x);
  lds[lane] = (lane & (HALF - 1)) < rows ? mine : make_float2(0.f, 0.f);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int BITS, int PREC>
__device__ __forceinline__ void scores(const Loaded<BITS>& x, const float2* scales, int c, int g, const Op (&q)[2], float q_sum, f32x4 (&s)[2]) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    Op k[2];
    if (BITS == 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j / 4].u[j % 4] = x.k[b][j % (BITS / 2)];
    } else {
      float2 as = make_float2(0.f, 0.f);
      if (!PREC) as = scales[16 * b + c];
      constexpr int PER = 32 / BITS;  // codes of a word
#pragma unroll
      for (int i = 0; i < BITS / 2; ++i) {
        const auto w = codes_of<BITS == 16 ? 8 : BITS, PREC>(x.k[b][i]);
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
          const int j = (PER * i + e) / 2;
          k[j / 4].u[j % 4] = values<PREC>(code(w, e), code(w, e + 1), as.y, as.x, as.y, as.x);
        }
      }
    }
    s[b] = mfma(k[1], q[1], mfma(k[0], q[0], f32x4{0, 0, 0, 0}));
  }
  if constexpr (PREC == 1 && BITS < 16)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {  // scale * product + offset * (sum of the query)
        const f32x4 as = *reinterpret_cast<const f32x4*>(&scales[16 * b + 4 * g + i]);
        s[b][i] = __builtin_fmaf(as[1], s[b][i], as[0] * q_sum);
        s[b][i + 1] = __builtin_fmaf(as[3], s[b][i + 1], as[2] * q_sum);
      }
}

struct Running {
  float m, l, offset;
  f32x4 o[4];
};

// Scores in s to weights. The sums so far are moved to a new maximum only where some lane's scores pass the old one.
__device__ __forceinline__ void soften(f32x4 (&s)[2], float scale2, Running& r) {
  const float top = max_nn(max_nn(max_nn(s[0][0], s[0][1]), max_nn(s[0][2], s[0][3])), max_nn(max_nn(s[1][0], s[1][1]), max_nn(s[1][2], s[1][3])));
  if (__builtin_amdgcn_ballot_w64(top * scale2 > r.m)) {
    const float m = max_nn(row_max(top) * scale2, r.m);
    const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(r.m - m);
    r.m = m;
    r.l *= alpha, r.offset *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db) r.o[db] *= alpha;
  }
  const float ref = r.m == -INFINITY ? 0.f : r.m;  // nothing visible yet: keep the empty state
  float sum = 0;
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale2, -ref));
      sum += s[b][i];
    }
  r.l += sum;
}

// The values by their weights (in s), which enter the product as the sum of TERMS bf16 values.
template <int BITS, int PREC, int TERMS>
__device__ __forceinline__ void weigh(const Loaded<BITS>& x, const float2* scales, int g, const f32x4 (&s)[2], Running& r) {
  Op p[TERMS];
  f32x4 as[2][2];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      float p0 = s[b][i], p1 = s[b][i + 1];
      if (BITS < 16) as[b][i / 2] = *reinterpret_cast<const f32x4*>(&scales[HALF + 16 * b + 4 * g + i]);
      if constexpr (PREC == 1 && BITS < 16) {
        const f32x4 m = as[b][i / 2];
        r.offset = __builtin_fmaf(p0, m[0], r.offset);
        r.offset = __builtin_fmaf(p1, m[2], r.offset);
        p0 *= m[1], p1 *= m[3];
      }
      uint32_t t[TERMS];
      split_pair<TERMS>(p0, p1, t);
#pragma unroll
      for (int k = 0; k < TERMS; ++k) p[k].u[2 * b + i / 2] = t[k];
    }
  Codes<BITS == 16 ? 8 : BITS, PREC> w[2][4];
  if (BITS < 16)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[b][i] = codes_of<BITS == 16 ? 8 : BITS, PREC>(x.v[b][i][0]);
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    Op v;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t y;
        if (BITS == 16) {
          const uint32_t x0 = x.v[b][i][(db >> 1) % (BITS == 16 ? 2 : 1)], x1 = x.v[b][i + 1][(db >> 1) % (BITS == 16 ? 2 : 1)];
          y = db & 1 ? (x0 >> 16) | (x1 & 0xffff0000u) : (x0 & 0xffffu) | (x1 << 16);
        } else {
          const f32x4 m = as[b][i / 2];
          y = values<PREC>(code(w[b][i], db), code(w[b][i + 1], db), m[1], m[0], m[3], m[2]);
        }
        v.u[2 * b + i / 2] = y;
      }
#pragma unroll
    for (int t = TERMS - 1; t >= 0; --t) r.o[db] = mfma(v, p[t], r.o[db]);
  }
}

// A wave's query rows and what it needs of them everywhere.
struct Rows {
  Op q[2];
  float q_sum, scale2;
  int c, g, lane;
  float2* scales;  // LDS
};

// Half pages [at, end) of one width (2 u and 2 u + 1: unit u). The next one's keys are loaded when this one's are
// multiplied, its values when these are. (A loop over pages of any width has to move what was loaded to the registers
// that its branches share, and waits for it there. Whole pages at a time take 200 registers, two waves a SIMD.)
template <int BITS, int PREC, int TERMS, class PAGE>
__device__ __forceinline__ void attend_pages(int& at, int end, PAGE page, const Rows& w, Running& r) {
  if (at >= end) return;
  Loaded<BITS> x;
  Half u = page(at);
  load_keys<BITS>(u, w.c, w.g, x);
  load_vals<BITS>(u, w.c, w.g, x);
  for (;;) {
    const int rows = u.rows;
    const bool more = ++at < end;
    f32x4 s[2];
    if (BITS < 16) share_scales<BITS, PREC>(w.scales, w.lane, x.pair, rows);
    scores<BITS, PREC>(x, w.scales, w.c, w.g, w.q, w.q_sum, s);
    if (more) {
      u = page(at);
      load_keys<BITS>(u, w.c, w.g, x);
    }
    if (rows < HALF) {  // rows that are not there: no score, and values of zero, so that what they hold meets no p of zero
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool there = 16 * b + 4 * w.g + i < rows;
          s[b][i] = there ? s[b][i] : -INFINITY;
#pragma unroll
          for (int j = 0; j < (BITS == 16 ? 2 : 1); ++j) x.v[b][i][j] = there ? x.v[b][i][j] : 0u;
        }
    }
    soften(s, w.scale2, r);
    weigh<BITS, PREC, TERMS>(x, w.scales, w.g, s, r);
    if (!more) break;
    load_vals<BITS>(u, w.c, w.g, x);
  }
}

// What a workgroup keeps in LDS.
struct ShortShared {
  f32x4 o[4][16][17];  // [wave][row][element / 4], padded
  float2 scales[4][2 * HALF];
  float ml[4][16][2];
};

// A workgroup's part of the launch, of 256 threads: `index` is its record's number times the heads and its head.
template <int PREC, int TERMS>
__device__ __forceinline__ void short_rows(const dkv_paged_args& a, float* part_o, float2* part_ml, int index, ShortShared& lds) {
  auto& ml = lds.ml;
  auto& o = lds.o;
  auto& scales = lds.scales;
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  const int H = a.plan.heads, G = a.plan.q_heads / H, record = index / H, h = index % H;
  if (a.bounds && record >= plan[N_WORK]) return;
  const Work w = plan_record<Work>(plan, a.plan.at_work, record);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int row0 = w.block * SHORT_BLOCK, rows_here = min(SHORT_BLOCK, w.count * G - row0);
  const int row = row0 + min(c, rows_here - 1), m = row / G;  // this lane's query row, its token of the sequence
  const int m_first = row0 / G, m_last = (row0 + rows_here - 1) / G;
  Rows rw;
  query_ops(static_cast<const uint16_t*>(a.q) + (int64_t)(h * G + row - m * G) * a.q_head_stride + (int64_t)(w.token0 + m) * a.q_tok_stride,
            c < rows_here, g, rw.q);
  rw.q_sum = query_sum(rw.q);
  rw.scale2 = a.scale * LOG2E;
  rw.c = c, rw.g = g, rw.lane = lane;
  rw.scales = scales[wave];
  const Op (&q)[2] = rw.q;
  const float scale2 = rw.scale2;
  Running r;
  r.m = -INFINITY, r.l = r.offset = 0.f;
  for (int db = 0; db < 4; ++db) r.o[db] = f32x4{0, 0, 0, 0};
  const uint8_t* const base = static_cast<const uint8_t*>(a.arena);
  const int64_t grain = grain_bytes(a.plan.layers, H), sub = (int64_t)a.layer * 2 * H + h;
  auto page = [&](int i) {
    const Page pg = plan_record<Page>(plan, a.plan.at_pages, w.first_page + i / 2);
    const int bits = page_bits(pg.page), first = i % 2 * HALF;
    const uint8_t *k = base + (pg.page >> 2) * grain + sub * page_sub(bits), *v = k + (int64_t)H * page_sub(bits);
    Half u;
    u.rows = min(HALF, pg.rows - first);  // (none: a page of up to 32 tokens)
    u.k = k + first * 8 * bits, u.v = v + first * 8 * bits;
    u.scales = (lane < HALF ? k : v) + (TILE * 8 * bits + 8 * first + 8 * (lane & (HALF - 1)));
    return u;
  };
  // A wave takes a fourth of the units that follow each other, so that it meets few widths.
  const int u0 = w.u0 + (w.u1 - w.u0) * wave / 4, u1 = w.u0 + (w.u1 - w.u0) * (wave + 1) / 4;
  int at = 2 * u0;
  attend_pages<4, PREC, TERMS>(at, 2 * min(w.n4, u1), page, rw, r);
  attend_pages<8, PREC, TERMS>(at, 2 * min(w.n8, u1), page, rw, r);
  attend_pages<16, PREC, TERMS>(at, 2 * min(w.n_pages, u1), page, rw, r);
  bool bad = false;  // some new value that is infinite or NaN was taken for zero
  for (; at < 2 * u1; ++at) {  // new tokens, as they are, up to each query row's own
    const int first = (at - 2 * w.n_pages) * HALF, seen = min(HALF, m_last + 1 - first), high = min(seen, m + 1 - first);
    if (seen <= 0) break;
    const bool mixed = m_first + 1 - first < seen;
    Half u;
    u.k = static_cast<const uint8_t*>(a.k_new) + 2 * (h * a.kn_head_stride + (int64_t)(w.token0 + first) * a.kn_tok_stride);
    u.v = static_cast<const uint8_t*>(a.v_new) + 2 * (h * a.vn_head_stride + (int64_t)(w.token0 + first) * a.vn_tok_stride);
    u.k_stride = (uint32_t)(2 * a.kn_tok_stride), u.v_stride = (uint32_t)(2 * a.vn_tok_stride);  // (of a single row, whatever it is)
    u.rows = min(HALF, w.count - first);
    Loaded<16> x;
    load_keys<16, true>(u, c, g, x);
    load_vals<16, true>(u, c, g, x);
    f32x4 s[2];
    scores<16, PREC>(x, rw.scales, c, g, q, rw.q_sum, s);
    // Values that not every query row of the block sees are zero where they are infinite or NaN (a p of zero makes NaN of
    // them) and are added after all units; those that none sees are zero.
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * b + 4 * g + i;
        s[b][i] = key < high ? s[b][i] : -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t& y = x.v[b][i][j];
          y = key < seen ? y : 0u;
          const uint32_t keep = mixed ? (bad_bf16(y) ? 0u : 0xffffu) | (bad_bf16(y >> 16) ? 0u : 0xffff0000u) : 0xffffffffu;
          bad = bad || keep != 0xffffffffu;
          y &= keep;
        }
      }
    soften(s, scale2, r);
    weigh<16, PREC, TERMS>(x, rw.scales, g, s, r);
  }
  r.l = row_sum(r.l);
  r.offset = PREC == 1 ? row_sum(r.offset) : 0.f;
  // (rare) Infinite and NaN values with their weights computed again: those that were taken for zero, and in elements that became NaN all
  // that is seen, since an infinite value's product with a weight's lower terms, which may be zero or negative, makes NaN of infinity.
  uint32_t lost = 0;  // such elements, of rows whose scores are no NaN: bit 4 db + i
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) lost |= r.o[db][i] != r.o[db][i] && r.l == r.l ? 1u << (4 * db + i) : 0u;
  const bool again = __builtin_amdgcn_ballot_w64(lost != 0);
  if (__builtin_amdgcn_ballot_w64(bad) || again) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) r.o[db][i] = lost >> (4 * db + i) & 1 ? 0.f : r.o[db][i];
    bool packed = false;  // a packed row of values is infinite or NaN: its elements stay NaN
    for (int at = again ? 2 * u0 : max(2 * u0, 2 * w.n_pages); at < 2 * u1; ++at) {
      const int first = (at - 2 * w.n_pages) * HALF;
      const uint8_t *key, *value;  // a row's, from its elements 16 g on
      int64_t k_stride = 128, v_stride = 128;
      int rows;
      if (first < 0) {
        const Half u = page(at);
        key = u.k + 32 * g, value = u.v + 32 * g, rows = u.rows;
        if (at < 2 * w.n8) {
          const float2 as = *reinterpret_cast<const float2*>(u.scales);
          packed = packed || (lane >= HALF && lane - HALF < rows && !(fabsf(as.x) < INFINITY && fabsf(as.y) < INFINITY));
          continue;
        }
      } else {
        rows = min(HALF, m_last + 1 - first);
        if (!again && m_first + 1 - first >= rows) continue;  // seen by every row
        key = static_cast<const uint8_t*>(a.k_new) + 2 * (h * a.kn_head_stride + (int64_t)(w.token0 + first) * a.kn_tok_stride) + 32 * g;
        value = static_cast<const uint8_t*>(a.v_new) + 2 * (h * a.vn_head_stride + (int64_t)(w.token0 + first) * a.vn_tok_stride) + 32 * g;
        k_stride = 2 * a.kn_tok_stride, v_stride = 2 * a.vn_tok_stride;
      }
      for (int j = 0; j < rows; ++j, key += k_stride, value += v_stride) {
        float dot = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x4 y = reinterpret_cast<const u32x4*>(key)[i];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dot = __builtin_fmaf(bf16_lo(q[i].u[e]), bf16_lo(y[e]), __builtin_fmaf(bf16_hi(q[i].u[e]), bf16_hi(y[e]), dot));
        }
        const float p = __builtin_amdgcn_exp2f(row_sum(dot) * scale2 - r.m);
        if (first + j > m) continue;  // (of pages: negative)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x4 y = reinterpret_cast<const u32x4*>(value)[i];
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // elements 16 g + 8 i + 2 e + ... = 16 g + 4 (2 i + e / 2) + 2 (e % 2) + ...
            if (bad_bf16(y[e])) r.o[2 * (e % 2)][2 * i + e / 2] += p * bf16_lo(y[e]);
            if (bad_bf16(y[e] >> 16)) r.o[2 * (e % 2) + 1][2 * i + e / 2] += p * bf16_hi(y[e]);
          }
        }
      }
    }
    const bool keep = __builtin_amdgcn_ballot_w64(packed);
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)  // (no such value was found: the NaN comes from a score)
        if (lost >> (4 * db + i) & 1 && (keep || r.o[db][i] == 0.f)) r.o[db][i] = NAN;
  }
  if (g == 0) ml[wave][c][0] = r.m, ml[wave][c][1] = r.l;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[wave][c][4 * g + i] = f32x4{r.o[0][i], r.o[1][i], r.o[2][i], r.o[3][i]} + r.offset;
  __syncthreads();
  const int rr = threadIdx.x >> 4, e4 = threadIdx.x & 15;  // the four waves' rows, four elements a thread
  if (rr >= rows_here) return;
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k][rr][0]);
  const float ref = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  f32x4 y = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float f = __builtin_amdgcn_exp2f(ml[k][rr][0] - ref);
    l += f * ml[k][rr][1];
    y += f * o[k][rr][e4];
  }
  if (w.part < 0) {
    const int out_row = row0 + rr, tok = out_row / G;
    store4(a.out, a.out_dtype, (int64_t)(w.token0 + tok) * a.out_tok_stride + (int64_t)(h * G + out_row - tok * G) * a.out_head_stride + 4 * e4,
           y / l);
  } else {
    const int64_t to = (int64_t)(w.part + rr) * H + h;
    *reinterpret_cast<f32x4*>(part_o + to * D + 4 * e4) = y;
    if (e4 == 0) part_ml[to] = make_float2(top, l);
  }
}

}  // namespace few
}  // namespace paged
}  // namespace dkv
