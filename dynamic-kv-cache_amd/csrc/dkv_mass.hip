// Attention mass (gfx950): what every token of the history and the chunk receives of the queries' softmax,
//   mass(h, t) = sum over the query heads of h and the queries m of exp(s_mt - max_m) / sum_m,
// the weight by which a cache forgets tokens. Two launches over the keys alone: the first gives every query row
// its maximum and sum over ranges of units (64 keys), the second joins them and sums each key's column over all
// rows, so that no sum is shared between workgroups and the result does not depend on their order. A workgroup
// dequantizes a unit's keys once, as MFMA operands in LDS, and its waves take the 16-row query blocks in turn.
#include "dkv_rows.h"

namespace dkv {
namespace mass {

using namespace rows;

constexpr int GROUP = 192;        // query rows of a row group: 12 blocks, three a wave
constexpr int BLOCKS = GROUP / 64;  // 16-row blocks of a wave

struct MassArgs {
  int splits, row_groups;
  float2* part;      // [heads][splits][rows] maximum (base 2) and sum
  float* out;        // [heads] rows of out_stride
  int64_t out_stride;
  int accumulate;
};

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
// history does.
__host__ __device__ inline int split_count(int most, int units) { return units < most ? units : most; }

// A unit's keys as MFMA operands in LDS: [key block][term][half][lane], a wave a key block.
template <int TERMS>
struct Keys {
  Op op[4][TERMS][2][64];
};

template <int BITS, int PREC, int TERMS>
__device__ __forceinline__ void stage_unit(const UnitRows& u, int wave, int lane, Keys<TERMS>& keys) {
  KeyPiece<BITS> p;
  load_key<BITS>(u, 16 * wave + (lane & 15), lane >> 4, p);
  Op op[Terms<BITS, PREC>::K][2];
  key_ops<BITS, PREC>(p, op);
#pragma unroll
  for (int t = 0; t < TERMS; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (t < Terms<BITS, PREC>::K) keys.op[wave][t][i][lane] = op[t < Terms<BITS, PREC>::K ? t : 0][i];
      else keys.op[wave][t][i][lane].v = bf16x8{};
    }
}

template <int PREC, int TERMS>
__device__ __forceinline__ UnitRows stage(const dkv_attn_args& a, const History& v, int unit, int h, int wave, int lane,
                                          Keys<TERMS>& keys) {
  const UnitRows u = unit < v.n_tiles ? tile_rows(a, a.tiles[unit], v.past, h) : chunk_rows(a, unit - v.n_tiles, h);
  const int bits = __builtin_amdgcn_readfirstlane(u.bits);
  if (bits == 4) stage_unit<4, PREC, TERMS>(u, wave, lane, keys);
  else if (bits == 8) stage_unit<8, PREC, TERMS>(u, wave, lane, keys);
  else stage_unit<16, PREC, TERMS>(u, wave, lane, keys);
  return u;
}

// Scaled scores (base 2) of 16 rows against the unit's keys 16 b + 4 g + i, -inf where a key is not visible: row c is
// chunk row m, whose segment starts at `start`; first is the unit's first chunk row, or negative for history.
template <int TERMS>
__device__ __forceinline__ void score(const Keys<TERMS>& keys, const Op (&q)[2], const UnitRows& u, int first, int m, int start,
                                      float scale2, int lane, f32x4 (&s)[4]) {
  const int g = lane >> 4;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = TERMS - 1; t >= 0; --t) s[b] = mfma(keys.op[b][t][1][lane], q[1], mfma(keys.op[b][t][0][lane], q[0], s[b]));
  }
  const int low = first < 0 ? 0 : start - first, high = first < 0 ? u.high : min(u.high, m + 1 - first);
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * b + 4 * g + i;
      s[b][i] = row >= low && row < high ? s[b][i] * scale2 : -INFINITY;
    }
}

// Query row `row` (query head by query head, q_heads / heads * nq of a KV head).
__device__ __forceinline__ void query_row(const dkv_attn_args& a, int h, int row, int rows, int g, Op (&q)[2]) {
  const int r = min(row, rows - 1), G = a.q_heads / a.heads;
  query_ops(static_cast<const uint16_t*>(a.q) + (h * G + r / a.nq) * a.q_head_stride + r % a.nq * a.q_tok_stride, row < rows, g, q);
}

template <int PREC>
__global__ __launch_bounds__(256) void stats_kernel(dkv_attn_args a, MassArgs p) {
  constexpr int TERMS = PREC == 0 ? 1 : 3;
  __shared__ Keys<TERMS> keys;
  const History v = history_of(a);
  const int splits = split_count(p.splits, v.units);
  if ((int)blockIdx.x >= splits) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, h = blockIdx.y;
  const int rows = a.q_heads / a.heads * a.nq;
  Op q[BLOCKS][2];
  float top[BLOCKS], sum[BLOCKS];
  int at[BLOCKS], start[BLOCKS];
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {
    const int row = blockIdx.z * GROUP + (4 * k + wave) * 16 + c;
    query_row(a, h, row, rows, g, q[k]);
    at[k] = row % a.nq, start[k] = chunk_seg_start(a, row % a.nq);
    top[k] = -INFINITY, sum[k] = 0.f;
  }
  const float scale2 = a.scale * LOG2E;
  const int from = (int)((int64_t)v.units * blockIdx.x / splits), to = (int)((int64_t)v.units * (blockIdx.x + 1) / splits);
  for (int unit = from; unit < to; ++unit) {
    __syncthreads();
    const UnitRows u = stage<PREC, TERMS>(a, v, unit, h, wave, lane, keys);
    __syncthreads();
    const int first = unit < v.n_tiles ? -1 : (unit - v.n_tiles) * TILE;
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
      // (a block none of whose rows sees a key of this chunk piece has nothing to add)
      if (first >= 0 && !__any(at[k] >= first && start[k] < first + TILE)) continue;
      f32x4 s[4];
      score<TERMS>(keys, q[k], u, first, at[k], start[k], scale2, lane, s);
      float m = top[k];
#pragma unroll
      for (int b = 0; b < 4; ++b) m = fmaxf(m, fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
      const float ref = m == -INFINITY ? 0.f : m;
      float l = sum[k] * __builtin_amdgcn_exp2f(top[k] - ref);
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(s[b][i] - ref);
      top[k] = m, sum[k] = l;
    }
  }
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {  // the four lanes of a row join theirs
    const float m = row_max(top[k]);
    const float l = row_sum(sum[k] * __builtin_amdgcn_exp2f(top[k] - (m == -INFINITY ? 0.f : m)));
    const int row = blockIdx.z * GROUP + (4 * k + wave) * 16 + c;
    if (g == 0 && row < rows) p.part[((int64_t)h * splits + blockIdx.x) * rows + row] = make_float2(m, l);
  }
}

template <int PREC>
__global__ __launch_bounds__(256) void columns_kernel(dkv_attn_args a, MassArgs p) {
  constexpr int TERMS = PREC == 0 ? 1 : 3;
  __shared__ Keys<TERMS> keys;
  __shared__ float2 norm[GROUP];  // maximum and 1 / sum of the row group's rows
  __shared__ float column[4][TILE];
  const History v = history_of(a);
  const int unit = blockIdx.x, h = blockIdx.y;
  if (unit >= v.units) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int rows = a.q_heads / a.heads * a.nq, splits = split_count(p.splits, v.units);
  const float scale2 = a.scale * LOG2E;
  const UnitRows u = stage<PREC, TERMS>(a, v, unit, h, wave, lane, keys);
  const int first = unit < v.n_tiles ? -1 : (unit - v.n_tiles) * TILE;
  float total[4][4] = {};
  for (int group = 0; group < p.row_groups; ++group) {
    __syncthreads();
    for (int i = threadIdx.x; i < GROUP; i += 256) {
      const int row = group * GROUP + i;
      float m = -INFINITY, l = 0.f;
      if (row < rows) {
        const float2* part = p.part + (int64_t)h * splits * rows + row;
        for (int s = 0; s < splits; ++s) m = fmaxf(m, part[(int64_t)s * rows].x);
        const float ref = m == -INFINITY ? 0.f : m;
        for (int s = 0; s < splits; ++s) l += part[(int64_t)s * rows].y * __builtin_amdgcn_exp2f(part[(int64_t)s * rows].x - ref);
      }
      norm[i] = row < rows ? make_float2(m, 1.f / l) : make_float2(0.f, 0.f);
    }
    __syncthreads();
    float sum[4][4] = {};  // this group's share, so that long sums are sums of short ones
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
      const int i = (4 * k + wave) * 16 + c, row = group * GROUP + i;
      if (group * GROUP + (4 * k + wave) * 16 >= rows) break;
      const int m = row % a.nq, start = chunk_seg_start(a, m);
      if (first >= 0 && !__any(m >= first && start < first + TILE)) continue;
      Op q[2];
      query_row(a, h, row, rows, g, q);
      f32x4 s[4];
      score<TERMS>(keys, q, u, first, m, start, scale2, lane, s);
      const float2 n = norm[i];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          // (a masked key gets nothing, also of a row whose sum is not a number)
          if (first < 0 || s[b][j] != -INFINITY) sum[b][j] += __builtin_amdgcn_exp2f(s[b][j] - n.x) * n.y;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) total[b][j] += sum[b][j];
  }
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // over the 16 rows of a block
      float x = total[b][j];
#pragma unroll
      for (int d = 8; d; d >>= 1) x += __shfl_xor(x, d, 16);
      if (c == 0) column[wave][16 * b + 4 * g + j] = x;
    }
  __syncthreads();
  const int key = threadIdx.x;
  if (key >= TILE || key >= u.high) return;
  const int token = unit < v.n_tiles ? a.tiles[unit].token_start + key : v.past + first + key;
  const float x = column[0][key] + column[1][key] + (column[2][key] + column[3][key]);
  float* out = p.out + h * p.out_stride + token;
  *out = p.accumulate ? *out + x : x;
}

constexpr int WORKGROUPS = 512;  // workgroups of the first launch
constexpr int MAX_SPLITS = 64;   // and the ranges of units that the second one joins, at most

static MassArgs plan_of(const dkv_attn_args& a) {
  MassArgs p{};
  const int64_t rows = (int64_t)(a.q_heads / a.heads) * a.nq;
  p.row_groups = (int)((rows + GROUP - 1) / GROUP);
  int64_t most = WORKGROUPS / ((int64_t)a.heads * p.row_groups);
  most = most < 1 ? 1 : most > MAX_SPLITS ? MAX_SPLITS : most;
  p.splits = split_count((int)most, a.n_tiles + (a.nq + TILE - 1) / TILE);
  return p;
}

static int64_t bytes_of(const dkv_attn_args& a, const MassArgs& p) {
  return (int64_t)a.heads * p.splits * (a.q_heads / a.heads) * a.nq * sizeof(float2);
}

}  // namespace mass

int check_history_args(const dkv_attn_args& a, const char* what);

}  // namespace dkv

using namespace dkv;
using namespace dkv::mass;

extern "C" {

int64_t dkv_attention_mass_workspace_bytes(const dkv_attn_args* args) {
  if (!args || args->heads <= 0 || args->q_heads <= 0 || args->q_heads % args->heads || args->nq <= 0 || args->n_tiles < 0) return 0;
  return bytes_of(*args, mass::plan_of(*args));
}

int dkv_attention_mass(const dkv_attn_args* args, float* mass, int64_t mass_head_stride, int32_t accumulate, void* stream) {
  clear_error();
  if (!args || !mass) {
    set_error("dkv_attention_mass: null args");
    return DKV_EINVAL;
  }
  const dkv_attn_args& a = *args;
  if (int rc = check_history_args(a, "dkv_attention_mass")) return rc;
  MassArgs p = mass::plan_of(a);
  if (p.row_groups > 65535 || (int64_t)(a.q_heads / a.heads) * a.nq > INT32_MAX - GROUP) {
    set_error("dkv_attention_mass: at most %d query rows a KV head", 65535 * GROUP);
    return DKV_EINVAL;
  }
  if (mass_head_stride < (int64_t)a.past + a.nq) {
    set_error("dkv_attention_mass: rows of %lld masses cannot hold %d tokens", (long long)mass_head_stride, a.past + a.nq);
    return DKV_EINVAL;
  }
  const int64_t need = bytes_of(a, p);
  if (!a.workspace || a.workspace_bytes < need) {
    set_error("dkv_attention_mass: workspace of %lld bytes needed, %lld given", (long long)need, (long long)a.workspace_bytes);
    return DKV_EINVAL;
  }
  p.part = static_cast<float2*>(a.workspace);
  p.out = mass, p.out_stride = mass_head_stride, p.accumulate = accumulate;
  const dim3 first(p.splits, a.heads, p.row_groups), second(a.n_tiles + (a.nq + TILE - 1) / TILE, a.heads);
  const hipStream_t st = (hipStream_t)stream;
  if (a.precision == 1) {
    hipLaunchKernelGGL(stats_kernel<1>, first, dim3(256), 0, st, a, p);
    hipLaunchKernelGGL(columns_kernel<1>, second, dim3(256), 0, st, a, p);
  } else {
    hipLaunchKernelGGL(stats_kernel<0>, first, dim3(256), 0, st, a, p);
    hipLaunchKernelGGL(columns_kernel<0>, second, dim3(256), 0, st, a, p);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
