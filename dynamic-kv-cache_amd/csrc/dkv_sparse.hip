// Sparse attention over the tiles that a cheap score selects for each query (gfx950).
//
// The index holds the elementwise smallest and largest key of every tile, so
//   score(h, m, t) = sum over the query heads of h and over d of max(q_d low_td, q_d high_td)
// bounds the sum of a query's scores over the tile's keys. As max(q x, q y) is q+ y + q- x for x <= y, with
// q+ = max(q, 0) and q- = min(q, 0), the sum over the query heads comes before the product: one dot product of
// 128 elements for each (query, KV head, tile). A query attends to the `blocks` tiles of the highest scores
// (equal ones: the first), to every tile after the index and to its chunk: scores and choice in one launch where the
// index is short (near_kernel), in two where it is long, then the attention, and a merge where a query's tiles are split
// over workgroups. Nothing of the history but the index, the chosen tiles and the tail is read.
//
// Measured (kernel times, 5 KV heads of 3 query heads unless said): a token past 8128 near 6.5, attention 6.2, merge
// 3.0 us, 16.7 us a call; a token past 131007 with 8 KV heads of 4 scores 4.4, choice 5.7, attention 6.2, merge 4.0, 20.3
// a call: latency, each launch a few dependent loads. 64 queries past 32704: 10.3 + 30.4 + 4.1, 42.2 a call; 513 queries
// past 20011 at fp32, 3 KV heads of 3: 22.4 + 8.4 + 101, 122 a call: every query walks some 30 tiles of its own and unpacks
// them, for three of 16 MFMA rows; the unpacking and the softmax keep the VALU busy, not the 400 MB from L2.
// Attention to all of a history is one launch and a merge, and reads each tile once for many queries: it is the faster one
// up to some length (a call of it and of this one at 16 blocks, us). One token, 5 KV heads of 3: 12.9 and 16.5 past 8128, 15.2
// and 17.0 past 32704, 21.6 and 21.2 past 65472, 32.2 and 21.2 past 131008; 8 of 4: 13.4 and 16.7, 16.9 and 16.8, 25.4 and
// 20.2, 42.2 and 20.2. 64 queries, 5 of 3: 16.1 and 29.3, 30.8 and 32.8, 48.6 and 40.2, 83.9 and 42.1.
#include "dkv_rows.h"
#include "dkv_select.h"

namespace dkv {
namespace sparse {

using namespace rows;

constexpr int BLOCK = 64;        // tiles of an index block
constexpr int BLOCK_PIECES = 16;  // 16-byte pieces of a tile's bounds: elements 8 p of low, then of high

// Index layout: [tile / 64][layer][head][16 pieces][64 tiles][8 bf16], so that lanes which hold a tile each read
// 1 KB of consecutive bytes, and an index that grows keeps its bytes in place.
__device__ __forceinline__ int64_t piece_at(int block, int layer, int layers, int h, int heads) {
  return (((int64_t)block * layers + layer) * heads + h) * BLOCK_PIECES * BLOCK;
}

// Tiles of an index workgroup, a wave a tile: 16 tiles' pieces of 16 bytes are 256 consecutive bytes of the index. Bound by
// the loads in flight, a tile's a wave: 32 layers of 5 heads past 8128 (97 MB) 36.5 us, 2.7 TB/s, half of what a large copy
// reaches; a workgroup a tile took 64.
constexpr int INDEX_TILES = 16;

// One step of a minimum (and maximum, of the negated) over lanes that halves the elements a lane holds: x keeps the lower
// half's lanes, y the upper half's. v_permlane swaps x's upper lanes with y's lower ones.
template <int LANES>
__device__ __forceinline__ void swap_lanes(float& x, float& y) {
  const auto r = LANES == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false)
                             : __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
}

// The bounds of a tile's keys, dequantized. Lane (row / 4, quarter): 16 elements of every 16th row; then halves of
// the elements change lanes, so that each lane ends with one element's bounds.
template <int BITS>
__device__ __forceinline__ void tile_bounds(const UnitRows& u, int lane, float& low, float& high) {
  float lo[16], hi[16];
  KeyPiece p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) load_key<BITS>(u, 16 * j + (lane >> 2), lane & 3, p[j]);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[j] = BITS == 16 ? (e & 1 ? bf16_hi(p[j].w[e / 2]) : bf16_lo(p[j].w[e / 2])) : code_at<BITS>(p[j].w, e) * p[j].as.y + p[j].as.x;
    lo[e] = fminf(fminf(fminf(x[0], x[1]), x[2]), x[3]);
    hi[e] = fmaxf(fmaxf(fmaxf(x[0], x[1]), x[2]), x[3]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    swap_lanes<32>(lo[e], lo[e + 8]), swap_lanes<32>(hi[e], hi[e + 8]);
    lo[e] = fminf(lo[e], lo[e + 8]), hi[e] = fmaxf(hi[e], hi[e + 8]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    swap_lanes<16>(lo[e], lo[e + 4]), swap_lanes<16>(hi[e], hi[e + 4]);
    lo[e] = fminf(lo[e], lo[e + 4]), hi[e] = fmaxf(hi[e], hi[e + 4]);
  }
#pragma unroll
  for (int half = 2, bit = 8; half >= 1; half >>= 1, bit >>= 1) {
    const bool upper = lane & bit;
#pragma unroll
    for (int e = 0; e < half; ++e) {
      const float give_lo = upper ? lo[e] : lo[e + half], give_hi = upper ? hi[e] : hi[e + half];
      const float got_lo = __shfl_xor(give_lo, bit, 64), got_hi = __shfl_xor(give_hi, bit, 64);
      lo[e] = fminf(upper ? lo[e + half] : lo[e], got_lo);
      hi[e] = fmaxf(upper ? hi[e + half] : hi[e], got_hi);
    }
  }
  low = lo[0], high = hi[0];
}

__global__ __launch_bounds__(64 * INDEX_TILES) void index_kernel(const uint8_t* arena, const dkv_tile* tiles, int tile0, int tile1,
                                                                 int layers, int heads, u32x4* bounds) {
  __shared__ u32x4 out[BLOCK_PIECES][INDEX_TILES];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int first = (tile0 / INDEX_TILES + blockIdx.x) * INDEX_TILES;
  const int layer = blockIdx.y / heads, h = blockIdx.y % heads;
  if (const int t = first + wave; t >= tile0 && t < tile1) {
    dkv_attn_args a{};
    a.arena = arena, a.layer = layer, a.heads = heads;
    const UnitRows u = tile_rows(a, tiles[t], INT32_MAX, h);
    const int bits = __builtin_amdgcn_readfirstlane(u.bits);
    float low, high;
    if (bits == 4) tile_bounds<4>(u, lane, low, high);
    else if (bits == 8) tile_bounds<8>(u, lane, low, high);
    else tile_bounds<16>(u, lane, low, high);
    const int d = 16 * (lane & 3) + 8 * (lane >> 5) + 4 * (lane >> 4 & 1) + 2 * (lane >> 3 & 1) + (lane >> 2 & 1);
    reinterpret_cast<uint16_t*>(&out[d / 8][wave])[d % 8] = (uint16_t)f32_to_bf16_rne(low);
    reinterpret_cast<uint16_t*>(&out[8 + d / 8][wave])[d % 8] = (uint16_t)f32_to_bf16_rne(high);
  }
  __syncthreads();
  if (threadIdx.x >= BLOCK_PIECES * INDEX_TILES) return;
  const int p = threadIdx.x / INDEX_TILES, i = threadIdx.x % INDEX_TILES, t = first + i;
  if (t >= tile0 && t < tile1) bounds[piece_at(t / BLOCK, layer, layers, h, heads) + p * BLOCK + t % BLOCK] = out[p][i];
}

// The history a launch sees: the arguments' or the device step's {past, n_tiles, n_indexed, single_rows}. A query attends
// to the `chosen` tiles of the index, to the `tiles` after it that are units of their own, and to the last single_rows
// tiles, of one 16-bit row each, 64 a unit: generated tokens, whose rows lie a slab apart.
struct Seen {
  int past, n_tiles, n_indexed, single_rows, chosen, tiles, singles;
};

__device__ __forceinline__ Seen seen_of(const dkv_attn_args& a, const dkv_sparse& s) {
  Seen v{a.past, a.n_tiles, s.n_indexed, s.single_rows};
  if (a.step) v = Seen{a.step[0], a.step[1], a.step[2], a.step[3]};
  v.n_indexed = min(min(v.n_indexed, s.n_indexed), v.n_tiles);
  v.single_rows = min(v.single_rows, v.n_tiles - v.n_indexed);
  v.chosen = min(s.blocks, v.n_indexed);
  v.tiles = v.n_tiles - v.n_indexed - v.single_rows;
  v.singles = (v.single_rows + TILE - 1) / TILE;
  return v;
}

struct SparsePlan {
  int row_blocks;          // 16-row blocks of a KV head's query heads
  int splits;              // workgroups of a (query, KV head, row block): as many as any history within the bounds takes
  int max_indexed, max_chosen;  // launch bounds
  int queries;             // that are scored at a time
  int64_t keys, lists, part_o, part_ml, bytes;  // workspace offsets
};

// Workgroups of a (query, KV head, row block): a unit a wave while `most` workgroups give room. Replays apply it to the
// history they find, with the launched workgroups as `most`, so they split it as a call over that history does.
__host__ __device__ inline int split_count(int most, int64_t units) {
  const int64_t want = (units + 3) / 4;
  return want < 1 ? 1 : want < most ? (int)want : most;
}
__device__ __forceinline__ int splits_of(const dkv_attn_args& a, const Seen& v, int most) {
  return split_count(most, (int64_t)v.chosen + v.tiles + v.singles + (a.nq + TILE - 1) / TILE);
}

constexpr int SCORE_QUERIES = 16;

// Scores of 64 tiles for 16 queries of a KV head, as sortable keys. Each wave takes 32 of the 128 elements, a lane
// a tile; their sums meet in LDS in a fixed order. In 64 bits, rounded to 32 at the end: the products of bf16 values
// are exact there and their sums as good as exact, so equal scores tie and no order of summation chooses a tile. Bound by
// these products: 513 queries by 520 tiles by 3 KV heads 22.4 us. Queries [first, first + some): a KV head's have `room`
// rows of keys.
__global__ __launch_bounds__(256) void score_kernel(dkv_attn_args a, dkv_sparse s, int max_indexed, int first, int room, uint32_t* keys) {
  __shared__ double query[SCORE_QUERIES][2 * D];  // q+ then q-, as the pieces' high and low
  __shared__ double part[4][SCORE_QUERIES][BLOCK];
  const Seen v = seen_of(a, s);
  const int block = blockIdx.x, h = blockIdx.y, m0 = first + blockIdx.z * SCORE_QUERIES;
  if (v.chosen == v.n_indexed || block * BLOCK >= v.n_indexed) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, G = a.q_heads / a.heads;
  const int queries = min(SCORE_QUERIES, a.nq - m0);
  constexpr int EACH = SCORE_QUERIES * D / 256, AHEAD = 4;  // sums a thread; query heads in flight
  double plus[EACH] = {}, minus[EACH] = {};
  const int d = threadIdx.x % D;
  for (int g0 = 0; g0 < G; g0 += AHEAD) {
    float x[AHEAD][EACH];
#pragma unroll
    for (int g = 0; g < AHEAD; ++g)
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int m = min(i * (256 / D) + (int)threadIdx.x / D, queries - 1);
        x[g][i] = bf16_lo((static_cast<const uint16_t*>(a.q) + (h * G + min(g0 + g, G - 1)) * a.q_head_stride + (m0 + m) * a.q_tok_stride)[d]);
      }
#pragma unroll
    for (int g = 0; g < AHEAD; ++g)
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (g0 + g < G) plus[i] += x[g][i] > 0.f ? x[g][i] : 0.f, minus[i] += x[g][i] > 0.f ? 0.f : x[g][i];
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int m = i * (256 / D) + (int)threadIdx.x / D;
    query[m][d] = minus[i];  // meets low
    query[m][D + d] = plus[i];
  }
  const u32x4* from = static_cast<const u32x4*>(s.bounds) + piece_at(block, a.layer, a.layers, h, a.heads) +
                      4 * wave * BLOCK + lane;
  double x[32];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const u32x4 w = block * BLOCK + lane < v.n_indexed ? from[p * BLOCK] : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) x[8 * p + 2 * j] = bf16_lo(w[j]), x[8 * p + 2 * j + 1] = bf16_hi(w[j]);
  }
  __syncthreads();
  for (int m = 0; m < queries; ++m) {
    double sum = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) sum = __builtin_fma(query[m][32 * wave + e], x[e], sum);
    part[wave][m][lane] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < queries * BLOCK; i += 256) {
    const int m = i / BLOCK, t = i % BLOCK;
    if (block * BLOCK + t < v.n_indexed)
      keys[((int64_t)h * room + m0 - first + m) * max_indexed + block * BLOCK + t] =
          order_key((float)(part[0][m][t] + part[1][m][t] + (part[2][m][t] + part[3][m][t])));
  }
}

// The chosen tiles of a (query, KV head), in order. Up to N * CHOOSERS keys stay in registers: a token past 131007 (2047
// tiles) 20.2 us a call with N = 8, 22.0 with keys loaded again each time (N = 0), which longer indexes take; 64 queries past
// 131007 50.9 and 52.8. Bound by the barriers of a radix step, about three a choice.
constexpr int CHOOSERS = 256;
template <int N>
__global__ __launch_bounds__(CHOOSERS) void choose_kernel(dkv_attn_args a, dkv_sparse s, int max_indexed, int max_chosen, int first,
                                                          int room, const uint32_t* keys, int32_t* lists) {
  __shared__ SelectScratch<CHOOSERS, 8> scratch;
  const Seen v = seen_of(a, s);
  if (v.chosen == v.n_indexed) return;  // every tile, or none: no list is read
  keys += ((int64_t)blockIdx.y * room + blockIdx.x) * max_indexed;
  lists += ((int64_t)blockIdx.y * a.nq + first + blockIdx.x) * max_chosen;
  auto key = [&](int i) { return max(keys[i], 1u); };
  Elements<CHOOSERS, N, decltype(key)>(v.n_indexed, key).largest(scratch, (uint32_t)v.chosen, [&](int to, int i) { lists[to] = i; });
}

// Scores and choice of a (query, KV head) in one workgroup, a wave 64 tiles: for up to NEAR_TILES indexed tiles. The sums
// are score_kernel's, term by term. Against scores and choice in two launches: a token past 8128 15.8 to 16.7 us a call and
// 19.6, past 32000 16.5 and 19.1, 64 queries past 32704 (511 tiles) 41.7 and 48.2. With room for 1024 tiles (1024 threads)
// one launch took longer than two above 512, 20.8 against 19.6 for a token past 65000 and 51.5 against 49.1 for 64 queries
// past 64000, and 47.1 at the 511.
constexpr int NEAR_TILES = 512;
__global__ __launch_bounds__(NEAR_TILES) void near_kernel(dkv_attn_args a, dkv_sparse s, int max_chosen, int32_t* lists) {
  __shared__ SelectScratch<NEAR_TILES, 8> scratch;
  __shared__ double query[2 * D];
  const Seen v = seen_of(a, s);
  if (v.chosen == v.n_indexed) return;
  const int m = blockIdx.x, h = blockIdx.y, G = a.q_heads / a.heads, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int tile = threadIdx.x;
  u32x4 w[BLOCK_PIECES];
  if (64 * wave < v.n_indexed) {
    const u32x4* from = static_cast<const u32x4*>(s.bounds) + piece_at(wave, a.layer, a.layers, h, a.heads) + lane;
#pragma unroll
    for (int p = 0; p < BLOCK_PIECES; ++p) w[p] = from[p * BLOCK];
  }
  if (threadIdx.x < D) {
    constexpr int AHEAD = 8;  // query heads in flight
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)h * G * a.q_head_stride + m * a.q_tok_stride + lane;
    double plus = 0, minus = 0;
    for (int g0 = 0; g0 < G; g0 += AHEAD) {
      float x[AHEAD];
#pragma unroll
      for (int g = 0; g < AHEAD; ++g) x[g] = bf16_lo(q[min(g0 + g, G - 1) * a.q_head_stride]);
#pragma unroll
      for (int g = 0; g < AHEAD; ++g)
        if (g0 + g < G) plus += x[g] > 0.f ? x[g] : 0.f, minus += x[g] > 0.f ? 0.f : x[g];
    }
    query[lane] = minus, query[D + lane] = plus;
  }
  __syncthreads();
  uint32_t mine = 0;
  if (64 * wave < v.n_indexed) {
    double part[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      part[k] = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const uint32_t x = w[4 * k + e / 8][e % 8 / 2];
        part[k] = __builtin_fma(query[32 * k + e], (double)(e & 1 ? bf16_hi(x) : bf16_lo(x)), part[k]);
      }
    }
    if (tile < v.n_indexed) mine = max(order_key((float)(part[0] + part[1] + (part[2] + part[3]))), 1u);
  }
  lists += ((int64_t)h * a.nq + m) * max_chosen;
  auto key = [&](int) { return mine; };  // (wave w's elements are the tiles from 64 w on)
  Elements<NEAR_TILES, 1, decltype(key)>(v.n_indexed, key).largest(scratch, (uint32_t)v.chosen, [&](int to, int i) { lists[to] = i; });
}

// A wave's running softmax over its units for 16 query rows: row c's maximum (base 2), this lane's share of its sum, of
// the packed rows' offsets in the output (precision 1), and the lane's 16 output elements.
struct Running {
  float m, l, offset;
  f32x4 o[4];
};

// p enters its product as the sum of TERMS bf16 values, so that only the values' own rounding limits a bf16 (two) or fp32
// (three) output. At precision 1 a packed row's scale goes into p, and its offset is summed beside.
template <int BITS, int PREC, int TERMS>
__device__ __forceinline__ void attend_unit(const UnitRows& u, const Op (&q)[2], float q_sum, float scale2, int c, int g, Running& r) {
  KeyPiece kp[4];
  ValuePiece<BITS> vp;
  f32x4 k_as[4][2], v_as[4][2];
#pragma unroll
  for (int b = 0; b < 4; ++b) load_key<BITS>(u, 16 * b + c, g, kp[b]);
  if (AFFINE<BITS, PREC>) load_scales<BITS>(u.k, u.rows, g, k_as);
  load_values<BITS>(u, c, g, vp);
  if (BITS < 16) load_scales<BITS>(u.v, u.rows, g, v_as);
  f32x4 s[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    Op k[2];
    key_ops<BITS, PREC>(kp[b], k);
    s[b] = mfma(k[1], q[1], mfma(k[0], q[0], f32x4{0, 0, 0, 0}));
  }
  if constexpr (AFFINE<BITS, PREC>) affine_scores<BITS>(k_as, q_sum, s);
  if (!__builtin_amdgcn_readfirstlane(u.low == 0 && u.high == TILE)) {
    // (A branch: masks of every element beside 64-bit row offsets took 136 us against 101, 513 queries past 20011.) Rows that are not visible: no score, and values of zero, so that what they hold (NaN or infinity) meets no p of zero.
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * b + 4 * g + i;
        const bool seen = row >= u.low && row < u.high;
        s[b][i] = seen ? s[b][i] : -INFINITY;
#pragma unroll
        for (int j = 0; j < (BITS == 16 ? 2 : 1); ++j) vp.w[b][i][j] = seen ? vp.w[b][i][j] : 0u;
        if (BITS < 16)
#pragma unroll
          for (int j = 0; j < 2; ++j) v_as[b][i / 2][2 * (i % 2) + j] = seen ? v_as[b][i / 2][2 * (i % 2) + j] : 0.f;
      }
  }
  float top = -INFINITY;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[b][i] *= scale2;
      top = fmaxf(top, s[b][i]);
    }
  top = fmaxf(row_max(top), r.m);
  const float ref = top == -INFINITY ? 0.f : top;  // nothing visible yet: keep the empty state
  const float alpha = __builtin_amdgcn_exp2f(r.m - ref);
  r.m = top;
  float sum = 0, offset = 0;
  Op p[TERMS][2];
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      float p0 = __builtin_amdgcn_exp2f(s[b][i] - ref), p1 = __builtin_amdgcn_exp2f(s[b][i + 1] - ref);
      sum += p0 + p1;
      if constexpr (AFFINE<BITS, PREC>) {
        const f32x4 m = v_as[b][i / 2];
        offset = __builtin_fmaf(p0, __builtin_fmaf(m[1], CENTRE<BITS>, m[0]), offset);
        offset = __builtin_fmaf(p1, __builtin_fmaf(m[3], CENTRE<BITS>, m[2]), offset);
        p0 *= m[1], p1 *= m[3];
      }
      uint32_t t[TERMS];
      split_pair<TERMS>(p0, p1, t);
#pragma unroll
      for (int k = 0; k < TERMS; ++k) p[k][b / 2].u[2 * (b % 2) + i / 2] = t[k];
    }
  r.l = r.l * alpha + sum;
  if (PREC == 1) r.offset = r.offset * alpha + offset;
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    Op v[2];
    value_ops<BITS, PREC>(vp, v_as, db, v);
    f32x4 o = r.o[db] * alpha;
#pragma unroll
    for (int t = TERMS - 1; t >= 0; --t) o = mfma(v[1], p[t][1], mfma(v[0], p[t][0], o));
    r.o[db] = o;
  }
}

__device__ __forceinline__ void store4(void* out, int out_dtype, int64_t at, f32x4 x) {
  if (out_dtype == 1)
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = x;
  else
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + at) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
}

// A wave a unit of 64 keys, keys and values straight from global memory into MFMA operands: a unit is read by one query
// alone, so LDS would only add a pass. 198 to 208 registers, two waves a SIMD; held to three they spilled (66 us against 54
// for 64 queries past 32704, then).
template <int PREC, int TERMS>
__global__ __launch_bounds__(256) void attend_kernel(dkv_attn_args a, dkv_sparse s, int row_blocks, int most, int max_chosen,
                                                     const int32_t* lists, float* part_o, float2* part_ml) {
  __shared__ float ml[4][16][2];
  __shared__ f32x4 o[4][16][17];  // [wave][row][element / 4], padded
  const Seen v = seen_of(a, s);
  const int splits = splits_of(a, v, most);
  if ((int)blockIdx.x >= splits) return;
  const int G = a.q_heads / a.heads, h = blockIdx.y / row_blocks, rb = blockIdx.y % row_blocks, m = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int heads_here = min(16, G - 16 * rb);
  const int64_t pair = (int64_t)h * a.nq + m;
  Op q[2];
  query_ops(static_cast<const uint16_t*>(a.q) + (h * G + 16 * rb + min(c, heads_here - 1)) * a.q_head_stride + m * a.q_tok_stride,
            c < heads_here, g, q);
  Running r;
  r.m = -INFINITY, r.l = r.offset = 0.f;
  const float q_sum = query_sum(q);
  for (int db = 0; db < 4; ++db) r.o[db] = f32x4{0, 0, 0, 0};
  const int start = chunk_seg_start(a, m), own_tile = v.chosen + v.tiles, history = own_tile + v.singles;
  const int piece0 = start / TILE, units = history + m / TILE - piece0 + 1;
  const bool listed = v.chosen < v.n_indexed;
  const float scale2 = a.scale * LOG2E;
  auto tile_at = [&](int i) {  // unit i's (first) tile, any that can be read where it is a chunk piece
    const int j = min(i, history - 1);
    if (j >= own_tile) return a.tiles[v.n_tiles - v.single_rows + TILE * (j - own_tile)];
    return a.tiles[j >= v.chosen ? v.n_indexed + j - v.chosen : listed ? lists[pair * max_chosen + j] : j];
  };
  int i = blockIdx.x * 4 + wave;
  dkv_tile t = {};
  if (history > 0) t = tile_at(i);
  for (; i < units; i += 4 * splits) {
    UnitRows u;
    if (i < history) {
      u = tile_rows(a, t, v.past, h);
      if (i >= own_tile) {
        u.rows = u.high = min(TILE, v.single_rows - TILE * (i - own_tile));
        u.k_stride = u.v_stride = (uint32_t)slab_bytes(1, 16, a.layers, a.heads);
      }
      t = tile_at(i + 4 * splits);  // the next unit's, while this one is computed
    } else {
      const int piece = piece0 + i - history;
      u = chunk_rows(a, piece, h);
      u.low = max(0, start - piece * TILE);
      u.high = min(TILE, m + 1 - piece * TILE);
    }
    const int bits = __builtin_amdgcn_readfirstlane(u.bits);
    if (bits == 4) attend_unit<4, PREC, TERMS>(u, q, q_sum, scale2, c, g, r);
    else if (bits == 8) attend_unit<8, PREC, TERMS>(u, q, q_sum, scale2, c, g, r);
    else attend_unit<16, PREC, TERMS>(u, q, q_sum, scale2, c, g, r);
  }
  r.l = row_sum(r.l);
  r.offset = PREC == 1 ? row_sum(r.offset) : 0.f;
  if (g == 0) ml[wave][c][0] = r.m, ml[wave][c][1] = r.l;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[wave][c][4 * g + i] = f32x4{r.o[0][i], r.o[1][i], r.o[2][i], r.o[3][i]} + r.offset;
  __syncthreads();
  const int row = threadIdx.x >> 4, e4 = threadIdx.x & 15;  // the four waves' rows, four elements a thread
  if (row >= heads_here) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][row][0]);
  const float ref = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  f32x4 x = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(ml[w][row][0] - ref);
    l += f * ml[w][row][1];
    x += f * o[w][row][e4];
  }
  if (gridDim.x == 1) {
    store4(a.out, a.out_dtype, m * a.out_tok_stride + (h * G + 16 * rb + row) * a.out_head_stride + 4 * e4, x / l);
  } else {
    const int64_t at = (pair * splits + blockIdx.x) * G + 16 * rb + row;
    *reinterpret_cast<f32x4*>(part_o + at * D + 4 * e4) = x;
    if (e4 == 0) part_ml[at] = make_float2(top, l);
  }
}

// Joins a query's splits: 16 lanes an output row, four elements a lane.
__global__ __launch_bounds__(256) void merge_kernel(dkv_attn_args a, dkv_sparse s, int most, const float* part_o,
                                                    const float2* part_ml) {
  const int G = a.q_heads / a.heads, row = blockIdx.x * 16 + (threadIdx.x >> 4), h = blockIdx.y, m = blockIdx.z;
  if (row >= G) return;
  const int splits = splits_of(a, seen_of(a, s), most), e4 = threadIdx.x & 15;
  const int64_t first = ((int64_t)h * a.nq + m) * splits * G + row;
  float top = -INFINITY;
  for (int i = e4; i < splits; i += 16) top = fmaxf(top, part_ml[first + (int64_t)i * G].x);
#pragma unroll
  for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 16));
  float l = 0.f;
  f32x4 x = {0, 0, 0, 0};
  constexpr int AHEAD = 8;  // splits in flight
  for (int i0 = 0; i0 < splits; i0 += AHEAD) {
    float2 p[AHEAD];
    f32x4 o[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t at = first + (int64_t)min(i0 + j, splits - 1) * G;
      p[j] = part_ml[at];
      o[j] = *reinterpret_cast<const f32x4*>(part_o + at * D + 4 * e4);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float f = i0 + j < splits ? __builtin_amdgcn_exp2f(p[j].x - top) : 0.f;
      l += f * p[j].y;
      x += f * o[j];
    }
  }
  store4(a.out, a.out_dtype, m * a.out_tok_stride + (h * G + row) * a.out_head_stride + 4 * e4, x / l);
}

// Bytes of scores at a time: a prompt of tens of thousands of queries over a long index would have gigabytes of them. (At
// least SCORE_QUERIES queries' whatever the index, and a multiple of these.)
constexpr int64_t KEYS_BYTES = 64 << 20;

// Attention workgroups that a call is split into: 64 queries past 32704 54 us with 1024, 62 with 512, 60 with 2048 (then).
constexpr int WORKGROUPS = 1024;

static SparsePlan plan_of(const dkv_attn_args& a, const dkv_sparse& s) {
  SparsePlan p{};
  const int G = a.q_heads / a.heads;
  p.row_blocks = (G + 15) / 16;
  p.max_indexed = s.n_indexed < a.n_tiles ? s.n_indexed : a.n_tiles;
  p.max_chosen = s.blocks < p.max_indexed ? s.blocks : p.max_indexed;
  const int64_t pairs = (int64_t)a.heads * a.nq;
  const int tail = a.n_tiles - p.max_indexed, single = a.step ? 0 : s.single_rows < tail ? s.single_rows : tail;
  int64_t units = (int64_t)p.max_chosen + tail - single + (single + TILE - 1) / TILE + (a.nq + TILE - 1) / TILE;
  if (a.step) units = (int64_t)a.n_tiles + (a.nq + TILE - 1) / TILE;  // a replay may find none of the tiles indexed
  const int64_t most = WORKGROUPS / (pairs * p.row_blocks);
  p.splits = split_count(most < 1 ? 1 : (int)most, units);
  auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  const int64_t choosing = p.max_chosen < p.max_indexed || a.step;
  p.keys = 0;
  p.queries = a.nq;
  int64_t scores = 0;  // (near_kernel keeps them in registers)
  if (choosing && p.max_indexed > NEAR_TILES) {
    const int64_t row = 4ll * a.heads * p.max_indexed, fit = KEYS_BYTES / row / SCORE_QUERIES * SCORE_QUERIES;
    if (fit < p.queries) p.queries = fit > SCORE_QUERIES ? (int)fit : SCORE_QUERIES < a.nq ? SCORE_QUERIES : a.nq;
    scores = row * p.queries;
  }
  p.lists = p.keys + up(scores);
  p.part_o = p.lists + (choosing ? up(4 * pairs * p.max_chosen) : 0);
  const int64_t parts = p.splits > 1 ? pairs * p.splits * G : 0;
  p.part_ml = p.part_o + up(4 * D * parts);
  p.bytes = p.part_ml + up(8 * parts);
  return p;
}

}  // namespace sparse

// What the sparse-attention and attention-mass calls ask of their arguments; `what` names the call.
int check_history_args(const dkv_attn_args& a, const char* what) {
  auto a16 = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  if (!a.q || !a.k_new || (a.n_tiles > 0 && (!a.tiles || !a.arena))) {
    set_error("%s: null pointer argument", what);
  } else if (a.heads <= 0 || a.q_heads <= 0 || a.q_heads % a.heads || a.nq <= 0 || a.past < 0 || a.n_tiles < 0 || a.layer < 0 ||
             a.layer >= a.layers || a.heads > 65535 / ((a.q_heads / a.heads + 15) / 16)) {
    set_error("%s: bad shape (heads %d, q_heads %d, nq %d, past %d, layer %d/%d)", what, a.heads, a.q_heads, a.nq, a.past,
              a.layer, a.layers);
  } else if (a.n_segs < 0 || a.n_segs > DKV_MAX_CHUNK_SEGS) {
    set_error("%s: n_segs %d outside [0, %d]", what, a.n_segs, DKV_MAX_CHUNK_SEGS);
  } else if (a.precision < 0 || a.precision > 1) {
    set_error("%s: precision must be 0 (bf16) or 1 (fp32)", what);
  } else if (!a16(a.q) || !a16(a.k_new) || (a.q_head_stride & 7) || (a.q_tok_stride & 7) || (a.kn_head_stride & 7) ||
             (a.kn_tok_stride & 7)) {
    set_error("%s: Q and K must be 16-byte aligned with strides that are multiples of 8 elements", what);
  } else if (a.nq > 1 && (a.kn_tok_stride < 0 || a.kn_tok_stride >= 1 << 23)) {
    set_error("%s: K's token stride must be from 0 to 2^23 - 1 elements", what);
  } else {
    if (a.n_segs <= 1) return 0;
    bool ok = a.seg_bounds[0] == 0 && a.seg_bounds[a.n_segs] == a.nq;
    for (int s = 0; s < a.n_segs; ++s) ok = ok && a.seg_bounds[s + 1] > a.seg_bounds[s];
    if (ok) return 0;
    set_error("%s: segment bounds must increase from 0 to nq", what);
  }
  return DKV_EINVAL;
}

}  // namespace dkv

using namespace dkv;
using namespace dkv::sparse;

extern "C" {

int64_t dkv_index_bytes(int32_t n_tiles, int32_t layers, int32_t heads) {
  if (n_tiles < 0 || layers <= 0 || heads <= 0) return 0;
  return ((int64_t)n_tiles + BLOCK - 1) / BLOCK * layers * heads * BLOCK_PIECES * BLOCK * 16;
}

int dkv_index(const void* arena, const dkv_tile* tiles, int32_t tile0, int32_t n_tiles, int32_t layers, int32_t heads,
              void* bounds, void* stream) {
  clear_error();
  if (tile0 < 0 || n_tiles < tile0 || layers <= 0 || heads <= 0 || (int64_t)layers * heads > 65535) {
    set_error("dkv_index: bad range (tiles [%d, %d), layers %d, heads %d)", tile0, n_tiles, layers, heads);
    return DKV_EINVAL;
  }
  if (n_tiles == tile0) return 0;
  if (!arena || !tiles || !bounds || ((uintptr_t)bounds & 15)) {
    set_error("dkv_index: null or misaligned pointer argument");
    return DKV_EINVAL;
  }
  const int groups = (n_tiles + INDEX_TILES - 1) / INDEX_TILES - tile0 / INDEX_TILES;
  hipLaunchKernelGGL(index_kernel, dim3(groups, layers * heads), dim3(64 * INDEX_TILES), 0, (hipStream_t)stream,
                     static_cast<const uint8_t*>(arena), tiles, tile0, n_tiles, layers, heads, static_cast<u32x4*>(bounds));
  return (int)hipGetLastError();
}

int64_t dkv_attend_sparse_workspace_bytes(const dkv_attn_args* args, const dkv_sparse* sparse) {
  if (!args || !sparse || args->heads <= 0 || args->q_heads <= 0 || args->q_heads % args->heads || args->nq <= 0 ||
      args->n_tiles < 0 || sparse->n_indexed < 0 || sparse->blocks < 0)
    return 0;
  return plan_of(*args, *sparse).bytes;
}

int dkv_attend_sparse(const dkv_attn_args* args, const dkv_sparse* sparse, void* stream) {
  clear_error();
  if (!args || !sparse) {
    set_error("dkv_attend_sparse: null args");
    return DKV_EINVAL;
  }
  const dkv_attn_args& a = *args;
  const dkv_sparse& s = *sparse;
  if (int rc = check_history_args(a, "dkv_attend_sparse")) return rc;
  if (!a.v_new || !a.out || ((uintptr_t)a.v_new & 15) || ((uintptr_t)a.out & 15) || (a.vn_head_stride & 7) ||
      (a.vn_tok_stride & 7) || (a.out_tok_stride & 3) || (a.out_head_stride & 3) || a.out_dtype < 0 || a.out_dtype > 1) {
    set_error("dkv_attend_sparse: V and out must be 16-byte aligned, strides multiples of 8 and 4 elements, out bf16 (0) or fp32 (1)");
    return DKV_EINVAL;
  }
  if (s.n_indexed < 0 || s.blocks < 0 || s.single_rows < 0 || (s.n_indexed > 0 && (!s.bounds || ((uintptr_t)s.bounds & 15)))) {
    set_error("dkv_attend_sparse: n_indexed %d, blocks %d and single_rows %d must not be negative, bounds 16-byte aligned", s.n_indexed,
              s.blocks, s.single_rows);
    return DKV_EINVAL;
  }
  if ((a.nq > 1 && (a.vn_tok_stride < 0 || a.vn_tok_stride >= 1 << 23)) || (int64_t)a.layers * a.heads > 65535) {
    set_error("dkv_attend_sparse: V's token stride must be from 0 to 2^23 - 1 elements, layers * heads at most 65535");
    return DKV_EINVAL;
  }
  if (a.nq > 65535) {
    set_error("dkv_attend_sparse: at most 65535 queries a call, got %d", a.nq);
    return DKV_EINVAL;
  }
  const SparsePlan p = plan_of(a, s);
  if (p.bytes > 0 && (!a.workspace || a.workspace_bytes < p.bytes)) {
    set_error("dkv_attend_sparse: workspace of %lld bytes needed, %lld given", (long long)p.bytes, (long long)a.workspace_bytes);
    return DKV_EINVAL;
  }
  const hipStream_t st = (hipStream_t)stream;
  char* ws = static_cast<char*>(a.workspace);
  uint32_t* keys = reinterpret_cast<uint32_t*>(ws + p.keys);
  int32_t* lists = reinterpret_cast<int32_t*>(ws + p.lists);
  float* part_o = reinterpret_cast<float*>(ws + p.part_o);
  float2* part_ml = reinterpret_cast<float2*>(ws + p.part_ml);
  if (p.max_chosen > 0 && (p.max_chosen < p.max_indexed || a.step)) {
    const int n = p.max_indexed;
    if (n <= NEAR_TILES) {
      hipLaunchKernelGGL(near_kernel, dim3(a.nq, a.heads), dim3(NEAR_TILES), 0, st, a, s, p.max_chosen, lists);
    } else {
      const auto choose = n <= 8 * CHOOSERS ? choose_kernel<8> : choose_kernel<0>;
      for (int m = 0; m < a.nq; m += p.queries) {
        const int some = a.nq - m < p.queries ? a.nq - m : p.queries;
        hipLaunchKernelGGL(score_kernel, dim3((n + BLOCK - 1) / BLOCK, a.heads, (some + SCORE_QUERIES - 1) / SCORE_QUERIES), dim3(256), 0, st,
                           a, s, n, m, p.queries, keys);
        hipLaunchKernelGGL(choose, dim3(some, a.heads), dim3(CHOOSERS), 0, st, a, s, n, p.max_chosen, m, p.queries, keys, lists);
      }
    }
  }
  const dim3 grid(p.splits, a.heads * p.row_blocks, a.nq);
  const auto attend = a.precision == 1 ? (a.out_dtype == 1 ? attend_kernel<1, 3> : attend_kernel<1, 2>)
                                       : (a.out_dtype == 1 ? attend_kernel<0, 3> : attend_kernel<0, 2>);
  hipLaunchKernelGGL(attend, grid, dim3(256), 0, st, a, s, p.row_blocks, p.splits, p.max_chosen, lists, part_o, part_ml);
  if (p.splits > 1)
    hipLaunchKernelGGL(merge_kernel, dim3((a.q_heads / a.heads + 15) / 16, a.heads, a.nq), dim3(256), 0, st, a, s, p.splits,
                       part_o, part_ml);
  return (int)hipGetLastError();
}

}  // extern "C"
