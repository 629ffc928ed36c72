// Attention mass (gfx950): what every token of the history and the chunk receives of the queries' softmax,
//   mass(h, t) = sum over the query heads of h and the queries m of exp(s_mt - max_m) / sum_m,
// the weight by which a cache forgets tokens. Two passes over the keys alone: the first gives every query row its
// maximum and sum over ranges of units (64 keys), the second joins them and sums each key's column over all rows. No
// sum is shared between workgroups, so the result does not depend on their order.
//   - up to 64 query rows a KV head (generated tokens): a wave a unit, keys and queries in registers, nothing in LDS. Of up
//     to 8 rows the first pass keeps the scores, and the second reads these alone;
//   - more: a workgroup a unit, whose waves unpack 16 keys each into MFMA operands in LDS and take the 16-row query
//     blocks in turn. The rows are joined in a launch between the passes, and where a chunk is long the second pass's
//     workgroups take a part of the rows each and one more launch adds the parts up.
// Measured (kernel times): a token past 131007 at fp32, 8 KV heads of 4: 29.9 us (73 MB of keys, 2.4 TB/s: two waves a SIMD
// wait for their next unit) + 8.5 (17 MB of scores). A 64-token frame past 8128, 5 KV heads of 3: 11.1 + 11.7, each a
// few dependent loads, three units a workgroup and the join. A 2048-token prompt past 1000: 29.9 + 4.9 + 42.1 + 4.8; the
// products alone are 6.7 us, each pass's 62 million exponentials with what surrounds them some 17 by counting instructions:
// no count explains what the passes take above that.
// Replays launch columns_kernel's workgroups for every tile that the table has room for, and those behind the history leave
// at once: attention and mass of a frame past 8128 36.7 us as calls, replayed 46.0 in a cache of 9152 tokens, 65.5 of
// 32768, 168.6 of 131072 (few_columns_kernel's grid is bounded: a token 19.0 to 20.3).
#include "dkv_rows.h"

namespace dkv {
namespace mass {

using namespace rows;

// Query rows of a KV head that a wave takes alone: what its registers hold (4 blocks of 16 rows, 255 at fp32), not where the
// two ways meet. A chunk of 48 rows past 8128 (5 KV heads) 13.0 us against 14.8 in workgroups, 63 rows 13.4 and 14.9; 64
// rows past 131007 at fp32 127 and 200, so there a 65th row costs more than half again.
constexpr int FEW = 64;
// Query rows of a KV head whose scores the first pass keeps for the second: a key's scores are 4 bytes a row written and
// read, its packed row 40 to 128 and the arithmetic again. A token over 131007 at fp32, 8 KV heads: 36.6 us with kept scores
// against 53.5 at 4 rows, 41.0 against 53.3 at 8. Room for 16 rows costs registers at every number of them: 52.2 us at 4, 63.4
// at 8, and 66.5, 74.6 and 86.5 at 9, 12 and 16, where none kept take 53.1 to 53.4.
constexpr int KEEP = 8;
constexpr int GROUP = 192;        // query rows of a row group: 12 blocks, three a wave
constexpr int BLOCKS = GROUP / 64;  // 16-row blocks of a wave

struct MassArgs {
  int splits, row_groups, row_parts;
  int kept;          // the scores stay for the second launch
  float2* part;      // [heads][splits][rows] maximum (base 2) and sum
  float2* norm;      // [heads][rows] reference and 1 / sum (many rows)
  float* columns;    // [row_parts][heads][stride] sums of a part of the rows (row_parts > 1); or with kept scores
                     // [heads][rows][stride] the scores, -infinity where masked
  int64_t columns_stride;
  float* out;        // [heads] rows of out_stride
  int64_t out_stride;
  int accumulate;
};

// Uniform to the compiler too: what a wave loops over stays in scalar registers, tiles come by scalar loads.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

struct History {
  int past, n_tiles, units;
};
__device__ __forceinline__ History history_of(const dkv_attn_args& a) {
  History v{a.past, a.n_tiles, 0};
  if (a.step) v.past = a.step[0], v.n_tiles = a.step[1];
  v.units = v.n_tiles + (a.nq + TILE - 1) / TILE;
  return v;
}

// Splits of the first launch that run for `units` units: replays split the history they find as a call over that
// history does. A workgroup of few rows has four units at a time.
__host__ __device__ inline int split_count(int most, int units, bool few) {
  const int want = few ? (units + 3) / 4 : units;
  return want < most ? want : most;
}

// A unit, and its first chunk row (negative for history).
struct Unit64 {
  UnitRows u;
  int first;
};
__device__ __forceinline__ Unit64 unit_of(const dkv_attn_args& a, const History& v, int unit, int h) {
  if (unit < v.n_tiles) return Unit64{tile_rows(a, a.tiles[unit], v.past, h), -1};
  return Unit64{chunk_rows(a, unit - v.n_tiles, h), (unit - v.n_tiles) * TILE};
}

// A row's scores are masked where the unit's key is not visible: keys [low, high) are. Row m's segment starts at `start`.
// Returns whether any is.
__device__ __forceinline__ bool mask_scores(const Unit64& x, int m, int start, int g, f32x4 (&s)[4]) {
  const int low = x.first < 0 ? 0 : start - x.first, high = x.first < 0 ? x.u.high : min(x.u.high, m + 1 - x.first);
  if (__all(low <= 0 && high >= TILE)) return false;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * b + 4 * g + i;
      if (row < low || row >= high) s[b][i] = -INFINITY;
    }
  return true;
}

// A row's maximum (raw) and sum with 16 scores more. The sum is of exp2(s * scale2 - reference), the reference being the
// maximum times scale2 as stored, so that both launches round it alike.
__device__ __forceinline__ void add_scores(const f32x4 (&s)[4], float scale2, float& top, float& sum) {
  float m = top;
#pragma unroll
  for (int b = 0; b < 4; ++b) m = fmaxf(m, fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
  const float ref = m == -INFINITY ? 0.f : m * scale2;
  float l = sum * __builtin_amdgcn_exp2f(top * scale2 - ref);
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale2, -ref));
  top = m, sum = l;
}

// Adds 16 keys' weights of a row (norm: reference and 1 / sum, 0 for a row that only fills a block up). A masked key gets
// nothing, also of a row whose sum is not a number.
template <bool MASKED>
__device__ __forceinline__ void add_weights(const f32x4 (&s)[4], float scale2, float2 norm, float (&sum)[4][4]) {
  if (norm.y == 0.f) return;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale2, -norm.x));
      const float x = __builtin_fmaf(p, norm.y, sum[b][i]);
      sum[b][i] = MASKED && s[b][i] == -INFINITY ? sum[b][i] : x;
    }
}

// A row's reference and sum with those of the splits [from, to).
constexpr int AHEAD = 16;  // loads in flight
__device__ __forceinline__ void join(const float2* part, int from, int to, int64_t stride, float& m, float& l) {
  for (int s0 = from; s0 < to; s0 += AHEAD) {
    float2 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = part[min(s0 + i, to - 1) * stride];
    float top = m;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, x[i].x);
    const float ref = top == -INFINITY ? 0.f : top;
    l *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) l += s0 + i < to ? x[i].y * __builtin_amdgcn_exp2f(x[i].x - ref) : 0.f;
    m = top;
  }
}

// A KV head's query rows lie query head by query head. The quotient of a row is below q_heads / heads <= 2^20, its product
// with the rounded 1 / nq off by less than one; put right after (an integer division a lane and block took a quarter of
// the second pass).
struct RowAt {
  int head, m;
};
__device__ __forceinline__ RowAt row_at(int row, int nq) {
  RowAt r;
  r.head = (int)((float)row * __builtin_amdgcn_rcpf((float)nq));
  r.m = (int)((uint32_t)row - (uint32_t)r.head * (uint32_t)nq);
  if (r.m < 0) --r.head, r.m += nq;
  if (r.m >= nq) ++r.head, r.m -= nq;
  return r;
}

// Query row `row`, the last one behind it (whose results are not used). Returns its query.
__device__ __forceinline__ int query_row(const dkv_attn_args& a, int h, int row, int rows, int g, Op (&q)[2]) {
  const RowAt r = row_at(min(row, rows - 1), a.nq);
  query_ops(static_cast<const uint16_t*>(a.q) + (h * (a.q_heads / a.heads) + r.head) * a.q_head_stride + r.m * a.q_tok_stride, true, g, q);
  return r.m;
}

// load_key of any width without a branch: what a branch loads is waited for where the widths meet, and the loads of a unit
// would come one after the other. Two pieces of 16 bytes always: at 8 bits the same one twice, at 4 bits one of which the
// second half lies in the next piece or in the scales (a sub-block has 8 bytes a row behind its codes).
struct __attribute__((packed, aligned(8))) Bytes16 {
  u32x4 x;
};
__device__ __forceinline__ void load_any(const UnitRows& u, int row, int g, KeyPiece& p) {
  const int r = row < u.rows ? row : 0;
  const uint8_t* at = u.k + (__umul24(r, u.k_stride) + g * 2 * u.bits);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4 x = reinterpret_cast<const Bytes16*>(at + (u.bits == 16 ? 16 * i : 0))->x;
#pragma unroll
    for (int j = 0; j < 4; ++j) p.w[4 * i + j] = x[j];
  }
  p.as = *reinterpret_cast<const float2*>(u.k + (u.bits == 16 ? 0 : u.rows * (8 * u.bits) + 8 * r));
}

// 16 sums a lane, [b][i] of key 16 b + 4 g + i, over the 16 lanes of a group: each lane ends with one key's, which it
// returns, and that key. Halves change places with the mirrored lane of 16, of 8, of 4 and of 2.
template <int CONTROL, int HALF>
__device__ __forceinline__ void fold(float (&x)[16], bool upper) {
#pragma unroll
  for (int i = 0; i < HALF; ++i) {
    const float give = upper ? x[i] : x[i + HALF], keep = upper ? x[i + HALF] : x[i];
    x[i] = keep + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), CONTROL, 0xf, 0xf, true));
  }
}
__device__ __forceinline__ float column_sum(const float (&sum)[4][4], int c, int g, int& key) {
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = sum[i / 4][i % 4];
  fold<0x140, 8>(x, c & 8);  // row_mirror
  fold<0x141, 4>(x, c & 4);  // row_half_mirror
  fold<0x1b, 2>(x, c & 2);   // quad_perm 3 2 1 0
  fold<0xb1, 1>(x, c & 1);   // quad_perm 1 0 3 2
  key = 16 * (c >> 2) + 4 * g + (c & 3);
  return x[0];
}

// ---- few rows: a wave a unit -----------------------------------------------------------------------------------
struct RawKeys {
  KeyPiece p[4];
  f32x4 as[4][2];
};

template <int PREC>
__device__ __forceinline__ void load_unit(const UnitRows& u, int c, int g, RawKeys& k) {
#pragma unroll
  for (int b = 0; b < 4; ++b) load_any(u, 16 * b + c, g, k.p[b]);
  if (PREC == 0) return;
  const uint8_t* scales = u.bits == 16 ? u.k : u.k + (int64_t)u.rows * (8 * u.bits);
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * b + 4 * g + 2 * i;
      k.as[b][i] = *reinterpret_cast<const f32x4*>(scales + (u.bits < 16 && row < u.rows ? 8 * row : 0));
    }
}

template <int BITS, int PREC, int NB>
__device__ __forceinline__ void unit_scores(const RawKeys& k, const Op (&q)[NB][2], const float (&q_sum)[NB], f32x4 (&s)[NB][4]) {
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    Op op[2];
    key_ops<BITS, PREC>(k.p[b], op);
#pragma unroll
    for (int n = 0; n < NB; ++n) s[n][b] = mfma(op[1], q[n][1], mfma(op[0], q[n][0], f32x4{0, 0, 0, 0}));
  }
  if constexpr (AFFINE<BITS, PREC>)
#pragma unroll
    for (int n = 0; n < NB; ++n) affine_scores<BITS>(k.as, q_sum[n], s[n]);
}

template <int PREC, int NB>
struct FewRows {
  Op q[NB][2];
  float q_sum[NB];
  int at[NB], start[NB];
  __device__ __forceinline__ void load(const dkv_attn_args& a, int h, int rows, int c, int g) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      at[n] = query_row(a, h, 16 * n + c, rows, g, q[n]);
      q_sum[n] = PREC == 1 ? query_sum(q[n]) : 0.f;
      start[n] = chunk_seg_start(a, at[n]);
    }
  }
  // use(unit, the unit, scores) of this wave's units unit, unit + step, ...: the next one's keys load meanwhile
  template <class Use>
  __device__ __forceinline__ void each(const dkv_attn_args& a, const History& v, int h, int unit, int step, int c, int g, Use use) {
    if (unit >= v.units) return;
    Unit64 x = unit_of(a, v, unit, h);
    x.u.bits = __builtin_amdgcn_readfirstlane(x.u.bits);
    RawKeys k;
    load_unit<PREC>(x.u, c, g, k);
    for (;;) {
      const int next = unit + step;
      Unit64 y = x;
      RawKeys l;
      if (next < v.units) {
        y = unit_of(a, v, next, h);
        y.u.bits = __builtin_amdgcn_readfirstlane(y.u.bits);
        load_unit<PREC>(y.u, c, g, l);
      }
      f32x4 s[NB][4];
      if (x.u.bits == 4) unit_scores<4, PREC, NB>(k, q, q_sum, s);
      else if (x.u.bits == 8) unit_scores<8, PREC, NB>(k, q, q_sum, s);
      else unit_scores<16, PREC, NB>(k, q, q_sum, s);
#pragma unroll
      for (int n = 0; n < NB; ++n) mask_scores(x, at[n], start[n], g, s[n]);
      use(unit, x, s);
      if (next >= v.units) return;
      unit = next, x = y, k = l;
    }
  }
};

// Kept scores are stored without a branch, lanes that have none behind the buffer's end, so that the next unit's loads,
// issued before, are waited for without the stores (51.9 us against 30 for a token over 131007 with branches).
constexpr uint32_t NOWHERE = 0xffffffffu;

template <int PREC, int NB>
__global__ __launch_bounds__(256) void few_stats_kernel(dkv_attn_args a, MassArgs p) {
  __shared__ float2 ml[4][16 * NB];
  const History v = history_of(a);
  const int splits = split_count(p.splits, v.units, true);
  if ((int)blockIdx.x >= splits) return;
  const int wave = wave_index(), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, h = blockIdx.y;
  const int rows = a.q_heads / a.heads * a.nq;
  FewRows<PREC, NB> few;
  few.load(a, h, rows, c, g);
  float top[NB], sum[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) top[n] = -INFINITY, sum[n] = 0.f;
  const float scale2 = a.scale * LOG2E;
  const auto kept = __builtin_amdgcn_make_buffer_rsrc(p.columns + (int64_t)h * rows * p.columns_stride, 0,
                                                      p.kept ? (int)(rows * p.columns_stride * 4) : 0, 0x00027000);
  few.each(a, v, h, 4 * blockIdx.x + wave, 4 * splits, c, g, [&](int unit, const Unit64& x, const f32x4 (&s)[NB][4]) {
#pragma unroll
    for (int n = 0; n < NB; ++n) add_scores(s[n], scale2, top[n], sum[n]);
    if (NB == 1 && p.kept) {
      const int token = x.first < 0 ? a.tiles[unit].token_start : v.past + x.first;
      const uint32_t row = 4u * (uint32_t)(c * p.columns_stride + token + 4 * g);
      if (x.u.high == TILE) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, s[0][b]), kept, c < rows ? row + 64 * b : NOWHERE, 0, 0);
      } else {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s[0][b][i]), kept,
                                                  c < rows && 16 * b + 4 * g + i < x.u.high ? row + 64 * b + 4 * i : NOWHERE, 0, 0);
      }
    }
  });
#pragma unroll
  for (int n = 0; n < NB; ++n) {  // the four lanes of a row join theirs
    const float m = row_max(top[n]), ref = m == -INFINITY ? 0.f : m * scale2;
    const float l = row_sum(sum[n] * __builtin_amdgcn_exp2f(top[n] * scale2 - ref));
    if (g == 0) ml[wave][16 * n + c] = make_float2(m * scale2, l);
  }
  __syncthreads();
  if ((int)threadIdx.x < rows) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][threadIdx.x].x);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < 4; ++w) l += ml[w][threadIdx.x].y * __builtin_amdgcn_exp2f(ml[w][threadIdx.x].x - ref);
    p.part[((int64_t)h * splits + blockIdx.x) * rows + threadIdx.x] = make_float2(m, l);
  }
}

// The rows' references and 1 / sum, joined from the splits by several threads a row; all threads call it.
template <int R>
struct Norms {
  static constexpr int SLICES = 256 / R;
  float2 ml[SLICES][R], norm[R];
  __device__ __forceinline__ void join_splits(const float2* part, int splits, int rows) {
    const int row = threadIdx.x % R, slice = threadIdx.x / R, from = splits * slice / SLICES, to = splits * (slice + 1) / SLICES;
    float m = -INFINITY, l = 0.f;
    if (row < rows) join(part + row, from, to, rows, m, l);
    ml[slice][row] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x < R) {
      m = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < SLICES; ++i) m = fmaxf(m, ml[i][threadIdx.x].x);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < SLICES; ++i) l += ml[i][threadIdx.x].y * __builtin_amdgcn_exp2f(ml[i][threadIdx.x].x - ref);
      norm[threadIdx.x] = (int)threadIdx.x < rows ? make_float2(m, 1.f / l) : make_float2(0.f, 0.f);
    }
    __syncthreads();
  }
};

template <int PREC, int NB>
__global__ __launch_bounds__(256) void few_columns_kernel(dkv_attn_args a, MassArgs p) {
  __shared__ Norms<16 * NB> norms;
  const History v = history_of(a);
  const int h = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  if (4 * (int)blockIdx.x >= v.units) return;
  const int rows = a.q_heads / a.heads * a.nq, splits = split_count(p.splits, v.units, true);
  FewRows<PREC, NB> few;
  few.load(a, h, rows, c, g);
  norms.join_splits(p.part + (int64_t)h * splits * rows, splits, rows);
  float2 nm[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) nm[n] = norms.norm[16 * n + c];
  const float scale2 = a.scale * LOG2E;
  few.each(a, v, h, 4 * blockIdx.x + wave, 4 * gridDim.x, c, g, [&](int unit, const Unit64& x, const f32x4 (&s)[NB][4]) {
    float sum[4][4] = {};
#pragma unroll
    for (int n = 0; n < NB; ++n) add_weights<true>(s[n], scale2, nm[n], sum);
    int key;
    const float w = column_sum(sum, c, g, key);
    if (key >= x.u.high) return;
    float* out = p.out + h * p.out_stride + (x.first < 0 ? a.tiles[unit].token_start : v.past + x.first) + key;
    *out = p.accumulate ? *out + w : w;
  });
}

// The columns of kept scores: EACH tokens a thread, no key and no tile is read again.
template <int EACH>
struct __attribute__((aligned(4 * EACH))) Scores {
  float x[EACH];
};
constexpr int EACH = 4;  // (a token a thread: 64.4 us against 58.9 for a token past 131007, more joins of the splits)
__global__ __launch_bounds__(256) void kept_columns_kernel(dkv_attn_args a, MassArgs p) {
  __shared__ Norms<16> norms;
  const History v = history_of(a);
  const int h = blockIdx.y, tokens = v.past + a.nq, token = (blockIdx.x * 256 + threadIdx.x) * EACH;
  if ((int)blockIdx.x * 256 * EACH >= tokens) return;
  const int rows = a.q_heads / a.heads * a.nq, splits = split_count(p.splits, v.units, true);
  Scores<EACH> s[KEEP];
  const float* from = p.columns + (int64_t)h * rows * p.columns_stride + min((int64_t)token, p.columns_stride - EACH);
#pragma unroll
  for (int r = 0; r < KEEP; ++r) s[r] = *reinterpret_cast<const Scores<EACH>*>(from + min(r, rows - 1) * p.columns_stride);
  norms.join_splits(p.part + (int64_t)h * splits * rows, splits, rows);
  const float scale2 = a.scale * LOG2E;
  float sum[EACH] = {};
#pragma unroll
  for (int r = 0; r < KEEP; ++r) {
    if (r >= rows) break;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r].x[i], scale2, -norms.norm[r].x));
      sum[i] = s[r].x[i] == -INFINITY ? sum[i] : __builtin_fmaf(w, norms.norm[r].y, sum[i]);
    }
  }
  float* out = p.out + h * p.out_stride + token;
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (token + i < tokens) out[i] = p.accumulate ? out[i] + sum[i] : sum[i];
}

// ---- many rows: a workgroup a unit -----------------------------------------------------------------------------
// A unit's keys as MFMA operands, a wave a 16-key block, and their (offset, scale) where scores take them.
struct Keys {
  Op op[4][2][64];
  f32x4 as[32];
};

template <int PREC>
__device__ __forceinline__ void stage_block(const UnitRows& u, const KeyPiece& p, int wave, int lane, Keys& keys) {
  Op op[2];
  if (u.bits == 4) key_ops<4, PREC>(p, op);
  else if (u.bits == 8) key_ops<8, PREC>(p, op);
  else key_ops<16, PREC>(p, op);
  keys.op[wave][0][lane] = op[0], keys.op[wave][1][lane] = op[1];
  if (PREC == 1 && lane < 16 && u.bits < 16) reinterpret_cast<float2*>(keys.as)[16 * wave + lane] = p.as;
}

template <int PREC>
__device__ __forceinline__ void block_scores(const Keys& keys, int bits, const Op (&q)[2], float q_sum, int lane, f32x4 (&s)[4]) {
  const int g = lane >> 4;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    s[b] = mfma(keys.op[b][1][lane], q[1], mfma(keys.op[b][0][lane], q[0], f32x4{0, 0, 0, 0}));
  if (PREC == 1 && bits < 16) {
    f32x4 as[4][2];
#pragma unroll
    for (int b = 0; b < 4; ++b) as[b][0] = keys.as[8 * b + 2 * g], as[b][1] = keys.as[8 * b + 2 * g + 1];
    if (bits == 4) affine_scores<4>(as, q_sum, s);
    else affine_scores<8>(as, q_sum, s);
  }
}

// (A chunk piece that no row of a block sees has nothing for it.)
__device__ __forceinline__ bool sees(const Unit64& x, int m, int start) {
  return x.first < 0 || __any(m >= x.first && start < x.first + TILE);
}

template <int PREC>
__global__ __launch_bounds__(256, PREC ? 2 : 4) void stats_kernel(dkv_attn_args a, MassArgs p) {
  __shared__ Keys keys;
  const History v = history_of(a);
  const int splits = split_count(p.splits, v.units, false);
  if ((int)blockIdx.x >= splits) return;
  const int wave = wave_index(), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, h = blockIdx.y;
  const int rows = a.q_heads / a.heads * a.nq;
  Op q[BLOCKS][2];
  float top[BLOCKS], sum[BLOCKS], q_sum[BLOCKS];
  int at[BLOCKS], start[BLOCKS];
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {
    const int row = blockIdx.z * GROUP + (4 * k + wave) * 16 + c;
    at[k] = query_row(a, h, row, rows, g, q[k]);
    q_sum[k] = PREC == 1 ? query_sum(q[k]) : 0.f;
    start[k] = chunk_seg_start(a, at[k]);
    top[k] = -INFINITY, sum[k] = 0.f;
  }
  const float scale2 = a.scale * LOG2E;
  // the units that the row group sees: up to its last query's
  const int first_row = blockIdx.z * GROUP, last_row = min(rows, first_row + GROUP) - 1;
  const RowAt r0 = row_at(first_row, a.nq), r1 = row_at(last_row, a.nq);
  const int last = r0.head == r1.head ? r1.m : a.nq - 1, units = v.n_tiles + last / TILE + 1;
  const int from = (int)((int64_t)units * blockIdx.x / splits), to = (int)((int64_t)units * (blockIdx.x + 1) / splits);
  Unit64 x = unit_of(a, v, from, h);
  x.u.bits = __builtin_amdgcn_readfirstlane(x.u.bits);
  KeyPiece piece;
  load_any(x.u, 16 * wave + c, g, piece);
  for (int unit = from; unit < to; ++unit) {
    __syncthreads();
    stage_block<PREC>(x.u, piece, wave, lane, keys);
    const Unit64 y = x;
    if (unit + 1 < to) {  // the next unit's keys load while this one's scores are computed
      x = unit_of(a, v, unit + 1, h);
      x.u.bits = __builtin_amdgcn_readfirstlane(x.u.bits);
      load_any(x.u, 16 * wave + c, g, piece);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
      if ((int)blockIdx.z * GROUP + (4 * k + wave) * 16 >= rows || !sees(y, at[k], start[k])) continue;
      f32x4 s[4];
      block_scores<PREC>(keys, y.u.bits, q[k], q_sum[k], lane, s);
      mask_scores(y, at[k], start[k], g, s);
      add_scores(s, scale2, top[k], sum[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {  // the four lanes of a row join theirs
    const float m = row_max(top[k]), ref = m == -INFINITY ? 0.f : m * scale2;
    const float l = row_sum(sum[k] * __builtin_amdgcn_exp2f(top[k] * scale2 - ref));
    const int row = blockIdx.z * GROUP + (4 * k + wave) * 16 + c;
    if (g == 0 && row < rows) p.part[((int64_t)h * splits + blockIdx.x) * rows + row] = make_float2(m * scale2, l);
  }
}

__global__ __launch_bounds__(256) void norm_kernel(dkv_attn_args a, MassArgs p) {
  const int rows = a.q_heads / a.heads * a.nq, row = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (row >= rows) return;
  const int splits = split_count(p.splits, history_of(a).units, false);
  float m = -INFINITY, l = 0.f;
  join(p.part + (int64_t)h * splits * rows + row, 0, splits, rows, m, l);
  p.norm[(int64_t)h * rows + row] = make_float2(m, 1.f / l);
}

// A wave's 16-row blocks come one after the other without a barrier, the next one's queries loading meanwhile.
struct QueryBlock {
  Op q[2];
  float2 norm;
  int m;
};
__device__ __forceinline__ QueryBlock load_query_block(const dkv_attn_args& a, const float2* norm, int h, int block, int rows, int c, int g) {
  QueryBlock x;
  const int row = 16 * block + c;
  x.m = query_row(a, h, row, rows, g, x.q);
  x.norm = norm[min(row, rows - 1)];
  if (row >= rows) x.norm = make_float2(0.f, 0.f);
  return x;
}

// JOIN: at most a row group, whose rows every workgroup joins itself (a launch less: a frame over 8128 22.2 us against
// 24.5).
template <int PREC, bool JOIN>
__global__ __launch_bounds__(256, PREC ? 2 : 4) void columns_kernel(dkv_attn_args a, MassArgs p) {
  __shared__ Keys keys;
  __shared__ float column[4][TILE];
  __shared__ float2 joined[JOIN ? GROUP : 1];
  const History v = history_of(a);
  const int unit = blockIdx.x, h = blockIdx.y;
  if (unit >= v.units) return;
  const int wave = wave_index(), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int rows = a.q_heads / a.heads * a.nq, blocks = (rows + 15) / 16;
  const int from = (int)((int64_t)blocks * blockIdx.z / p.row_parts), to = (int)((int64_t)blocks * (blockIdx.z + 1) / p.row_parts);
  const float scale2 = a.scale * LOG2E;
  Unit64 x = unit_of(a, v, unit, h);
  x.u.bits = __builtin_amdgcn_readfirstlane(x.u.bits);
  KeyPiece piece;
  load_any(x.u, 16 * wave + c, g, piece);
  if (JOIN && (int)threadIdx.x < rows) {
    const int splits = split_count(p.splits, v.units, false);
    float m = -INFINITY, l = 0.f;
    join(p.part + (int64_t)h * splits * rows + threadIdx.x, 0, splits, rows, m, l);
    joined[threadIdx.x % GROUP] = make_float2(m, 1.f / l);
  }
  stage_block<PREC>(x.u, piece, wave, lane, keys);
  __syncthreads();
  const float2* norm = JOIN ? joined : p.norm + (int64_t)h * rows;
  // the next block from `b` on of which a row may see the unit: queries come one after the other within a query head
  auto seeing = [&](int b) {
    for (; b < to; b += 4)
      if (const int m = row_at(16 * b, a.nq).m + 15; m >= x.first || m >= a.nq) break;
    return b;
  };
  int block = seeing(from + wave);
  QueryBlock now = load_query_block(a, norm, h, min(block, blocks - 1), rows, c, g);
  float total[4][4] = {};
  constexpr int SHORT = 8;  // blocks whose sums are added up before they join the total, so that long sums are sums of short ones
  while (block < to) {
    float sum[4][4] = {};
    for (int i = 0; i < SHORT && block < to; ++i) {
      const int after = seeing(block + 4);
      const QueryBlock next = load_query_block(a, norm, h, min(after, blocks - 1), rows, c, g);
      const int start = chunk_seg_start(a, now.m);
      if (sees(x, now.m, start)) {
        f32x4 s[4];
        block_scores<PREC>(keys, x.u.bits, now.q, PREC == 1 ? query_sum(now.q) : 0.f, lane, s);
        if (mask_scores(x, now.m, start, g, s)) add_weights<true>(s, scale2, now.norm, sum);
        else add_weights<false>(s, scale2, now.norm, sum);
      }
      now = next, block = after;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) total[b][j] += sum[b][j];
  }
  int key;
  const float w = column_sum(total, c, g, key);
  column[wave][key] = w;
  __syncthreads();
  key = threadIdx.x;
  if (key >= TILE || key >= x.u.high) return;
  const int token = (x.first < 0 ? a.tiles[unit].token_start : v.past + x.first) + key;
  const float all = column[0][key] + column[1][key] + (column[2][key] + column[3][key]);
  if (p.row_parts > 1) {
    p.columns[((int64_t)blockIdx.z * a.heads + h) * p.columns_stride + token] = all;
  } else {
    float* out = p.out + h * p.out_stride + token;
    *out = p.accumulate ? *out + all : all;
  }
}

__global__ __launch_bounds__(256) void add_parts_kernel(dkv_attn_args a, MassArgs p) {
  const int token = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (token >= history_of(a).past + a.nq) return;
  float x = 0.f;
  for (int i = 0; i < p.row_parts; ++i) x += p.columns[((int64_t)i * a.heads + h) * p.columns_stride + token];
  float* out = p.out + h * p.out_stride + token;
  *out = p.accumulate ? *out + x : x;
}

// Workgroups of a launch where there is work for as many, and ranges of units that the second launch joins, at most. Many
// rows: 2048 and 4096 workgroups took 78.0 and 82.2 us for 2048 tokens past 1000 against 77.9 with 1024. Few rows: 1024
// workgroups of up to 128 splits 66.6 us for a token past 131007 against 61.2 (two workgroups a CU are resident, and each
// joins the splits once).
constexpr int WORKGROUPS = 1024;
constexpr int MAX_SPLITS = 32;
constexpr int WORKGROUPS_FEW = 512;
constexpr int MAX_SPLITS_FEW = 64;
constexpr int MAX_ROW_PARTS = 8;  // 2048 tokens past 1000 74.9 us, with 4 parts 78.3, with 2 85.7, with 16 the same

struct MassPlan {
  MassArgs p;
  int64_t part_bytes, norm_bytes, bytes;
};

static MassPlan plan_of(const dkv_attn_args& a) {
  MassPlan m{};
  const int64_t rows = (int64_t)(a.q_heads / a.heads) * a.nq, units = (int64_t)a.n_tiles + (a.nq + TILE - 1) / TILE;
  m.p.row_groups = (int)((rows + GROUP - 1) / GROUP);
  const bool few = rows <= FEW;
  int64_t most = (few ? WORKGROUPS_FEW : WORKGROUPS) / ((int64_t)a.heads * m.p.row_groups);
  const int64_t cap = few ? MAX_SPLITS_FEW : MAX_SPLITS;
  most = most < 1 ? 1 : most > cap ? cap : most;
  m.p.splits = split_count((int)most, (int)units, few);
  // four row groups and more a part: by the chunk alone, so that replays add up what a call does
  m.p.row_parts = m.p.row_groups / 4;
  if (m.p.row_parts > MAX_ROW_PARTS) m.p.row_parts = MAX_ROW_PARTS;
  if (m.p.row_parts < 1) m.p.row_parts = 1;
  m.p.columns_stride = ((int64_t)a.past + a.nq + 63) & ~63;
  m.part_bytes = ((int64_t)a.heads * m.p.splits * rows * sizeof(float2) + 255) & ~(int64_t)255;
  m.norm_bytes = few ? 0 : ((int64_t)a.heads * rows * sizeof(float2) + 255) & ~(int64_t)255;
  m.p.kept = rows <= KEEP && rows * m.p.columns_stride * 4 <= INT32_MAX;
  const int64_t columns = m.p.kept ? rows : m.p.row_parts > 1 ? m.p.row_parts : 0;
  m.bytes = m.part_bytes + m.norm_bytes + columns * a.heads * m.p.columns_stride * 4;
  return m;
}

}  // namespace mass

int check_history_args(const dkv_attn_args& a, const char* what);

}  // namespace dkv

using namespace dkv;
using namespace dkv::mass;

extern "C" {

int64_t dkv_attention_mass_workspace_bytes(const dkv_attn_args* args) {
  if (!args || args->heads <= 0 || args->q_heads <= 0 || args->q_heads % args->heads || args->nq <= 0 || args->n_tiles < 0) return 0;
  return mass::plan_of(*args).bytes;
}

int dkv_attention_mass(const dkv_attn_args* args, float* mass, int64_t mass_head_stride, int32_t accumulate, void* stream) {
  clear_error();
  if (!args || !mass) {
    set_error("dkv_attention_mass: null args");
    return DKV_EINVAL;
  }
  const dkv_attn_args& a = *args;
  if (int rc = check_history_args(a, "dkv_attention_mass")) return rc;
  const MassPlan plan = mass::plan_of(a);
  MassArgs p = plan.p;
  const int64_t rows = (int64_t)(a.q_heads / a.heads) * a.nq;
  if (p.row_groups > 65535 || rows > INT32_MAX - GROUP) {
    set_error("dkv_attention_mass: at most %d query rows a KV head", 65535 * GROUP);
    return DKV_EINVAL;
  }
  if (mass_head_stride < (int64_t)a.past + a.nq) {
    set_error("dkv_attention_mass: rows of %lld masses cannot hold %d tokens", (long long)mass_head_stride, a.past + a.nq);
    return DKV_EINVAL;
  }
  if (!a.workspace || a.workspace_bytes < plan.bytes) {
    set_error("dkv_attention_mass: workspace of %lld bytes needed, %lld given", (long long)plan.bytes, (long long)a.workspace_bytes);
    return DKV_EINVAL;
  }
  p.part = static_cast<float2*>(a.workspace);
  p.norm = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + plan.part_bytes);
  p.columns = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + plan.part_bytes + plan.norm_bytes);
  p.out = mass, p.out_stride = mass_head_stride, p.accumulate = accumulate;
  const hipStream_t st = (hipStream_t)stream;
  const int units = a.n_tiles + (a.nq + TILE - 1) / TILE;
  if (rows <= FEW) {
    const auto stats = a.precision == 1 ? (rows <= 16 ? few_stats_kernel<1, 1> : few_stats_kernel<1, 4>)
                                        : (rows <= 16 ? few_stats_kernel<0, 1> : few_stats_kernel<0, 4>);
    const auto columns = a.precision == 1 ? (rows <= 16 ? few_columns_kernel<1, 1> : few_columns_kernel<1, 4>)
                                          : (rows <= 16 ? few_columns_kernel<0, 1> : few_columns_kernel<0, 4>);
    const int by_unit = (units + 3) / 4, most = WORKGROUPS_FEW / a.heads;
    hipLaunchKernelGGL(stats, dim3(p.splits, a.heads), dim3(256), 0, st, a, p);
    if (p.kept)
      hipLaunchKernelGGL(kept_columns_kernel, dim3((a.past + a.nq + 256 * EACH - 1) / (256 * EACH), a.heads), dim3(256), 0, st, a, p);
    else
      hipLaunchKernelGGL(columns, dim3(by_unit < most ? by_unit : most < 1 ? 1 : most, a.heads), dim3(256), 0, st, a, p);
    return (int)hipGetLastError();
  }
  const auto stats = a.precision == 1 ? stats_kernel<1> : stats_kernel<0>;
  const bool joins = p.row_groups == 1;
  const auto columns = a.precision == 1 ? (joins ? columns_kernel<1, true> : columns_kernel<1, false>)
                                        : (joins ? columns_kernel<0, true> : columns_kernel<0, false>);
  hipLaunchKernelGGL(stats, dim3(p.splits, a.heads, p.row_groups), dim3(256), 0, st, a, p);
  if (!joins) hipLaunchKernelGGL(norm_kernel, dim3((unsigned)((rows + 255) / 256), a.heads), dim3(256), 0, st, a, p);
  hipLaunchKernelGGL(columns, dim3(units, a.heads, p.row_parts), dim3(256), 0, st, a, p);
  if (p.row_parts > 1)
    hipLaunchKernelGGL(add_parts_kernel, dim3((a.past + a.nq + 255) / 256, a.heads), dim3(256), 0, st, a, p);
  return (int)hipGetLastError();
}

}  // extern "C"
