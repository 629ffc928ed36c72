// Attention of a step's new tokens over pages (gfx950).
#include "dkv_rows.h"
#include "dkv_paged.h"

namespace dkv {
namespace paged {

using namespace rows;

// A unit's rows: a page's, or 64 new tokens' from `k` and `v` on. Rows [0, rows) are there.
struct Unit {
  const uint8_t* k;
  const uint8_t* v;
  uint32_t k_stride, v_stride;  // bytes from row to row, below 2^24
  int bits, rows;
  int high;  // rows that this lane's query row sees
};

struct Running {
  float m, l, offset;
  f32x4 o[4];
};

template <int BITS>
__device__ __forceinline__ void load_page_key(const Unit& u, int row, int g, KeyPiece& p) {
  const int r = row < u.rows ? row : 0;
  const uint8_t* at = u.k + (__umul24(r, u.k_stride) + g * 2 * BITS);
  if (BITS == 4) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
    p.w[0] = w[0], p.w[1] = w[1];
  } else {
#pragma unroll
    for (int i = 0; i < BITS / 8; ++i) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(at + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) p.w[4 * i + j] = w[j];
    }
  }
  if (BITS < 16) p.as = *reinterpret_cast<const float2*>(u.k + (TILE * 8 * BITS + 8 * r));
}

// (offset, scale) of the lane's rows 16 b + 4 g + i, two rows a load.
template <int BITS>
__device__ __forceinline__ void load_page_scales(const uint8_t* base, int rows, int g, f32x4 (&as)[4][2]) {
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * b + 4 * g + 2 * i;
      as[b][i] = *reinterpret_cast<const f32x4*>(base + (TILE * 8 * BITS + 8 * (row < rows ? row : 0)));
    }
}

// New tokens that some rows of a block see and others do not, of which one has a value that is infinite or NaN: the
// products took zeros for these values, here they are added for the rows that see them. `p` is room for 16 x 64 floats.
__device__ __forceinline__ void add_bad_values(const Unit& u, int rows, const f32x4 (&e)[4], int c, int g, float* p, Running& r) {
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) p[c * TILE + 16 * b + 4 * g + i] = e[b][i];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  for (int j = 0; j < rows; ++j) {
    const uint32_t* v = reinterpret_cast<const uint32_t*>(u.v + __umul24(j, u.v_stride) + 32 * g);
    if (j >= u.high) continue;
    const float pj = p[c * TILE + j];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t w = v[k];
      if (bad_bf16(w)) r.o[(2 * k) % 4][k / 2] += pj * bf16_lo(w);
      if (bad_bf16(w >> 16)) r.o[(2 * k + 1) % 4][k / 2] += pj * bf16_hi(w);
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// `rows`: rows of the unit that some query row of the block sees; `mixed`: they do not all see the same ones.
template <int BITS, int PREC, int TERMS>
__device__ __forceinline__ void attend_unit(const Unit& u, int rows, bool mixed, const Op (&q)[2], float q_sum, float scale2, int c, int g,
                                            float* lds, Running& r) {
  KeyPiece kp[4];
  ValuePiece<BITS> vp;
  f32x4 k_as[4][2], v_as[4][2];
#pragma unroll
  for (int b = 0; b < 4; ++b) load_page_key<BITS>(u, 16 * b + c, g, kp[b]);
  if (AFFINE<BITS, PREC>) load_page_scales<BITS>(u.k, u.rows, g, k_as);
  load_values<BITS>(UnitRows{u.k, u.v, u.k_stride, u.v_stride, BITS, u.rows, 0, u.rows}, c, g, vp);
  if (BITS < 16) load_page_scales<BITS>(u.v, u.rows, g, v_as);
  f32x4 s[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    Op k[2];
    key_ops<BITS, PREC>(kp[b], k);
    s[b] = mfma(k[1], q[1], mfma(k[0], q[0], f32x4{0, 0, 0, 0}));
  }
  if constexpr (AFFINE<BITS, PREC>) affine_scores<BITS>(k_as, q_sum, s);
  bool bad = false;
  if (rows < TILE || mixed) {
    // Rows that are not visible: no score, and values of zero, so that what they hold (NaN or infinity) meets no p of zero.
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * b + 4 * g + i;
        s[b][i] = row < u.high ? s[b][i] : -INFINITY;
#pragma unroll
        for (int j = 0; j < (BITS == 16 ? 2 : 1); ++j) vp.w[b][i][j] = row < rows ? vp.w[b][i][j] : 0u;
        if (BITS < 16)
#pragma unroll
          for (int j = 0; j < 2; ++j) v_as[b][i / 2][2 * (i % 2) + j] = row < rows ? v_as[b][i / 2][2 * (i % 2) + j] : 0.f;
      }
    if (BITS == 16 && mixed) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) bad = bad || bad_bf16(vp.w[b][i][j % (BITS == 16 ? 2 : 1)]) || bad_bf16(vp.w[b][i][j % (BITS == 16 ? 2 : 1)] >> 16);
      bad = __builtin_amdgcn_ballot_w64(bad) != 0;
      if (bad)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t& w = vp.w[b][i][j % (BITS == 16 ? 2 : 1)];
              w &= (bad_bf16(w) ? 0u : 0xffffu) | (bad_bf16(w >> 16) ? 0u : 0xffff0000u);
            }
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
      s[b][i] = p0, s[b][i + 1] = p1;
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
  if (BITS == 16 && bad) add_bad_values(u, rows, s, c, g, lds, r);
}

template <int PREC, int TERMS>
__global__ __launch_bounds__(256) void short_kernel(dkv_paged_args a, float* part_o, float2* part_ml) {
  __shared__ float ml[4][16][2];
  __shared__ f32x4 o[4][16][17];  // [wave][row][element / 4], padded
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  const int H = a.plan.heads, G = a.plan.q_heads / H, record = blockIdx.x / H, h = blockIdx.x % H;
  if (a.bounds && record >= plan[N_WORK]) return;
  const Work w = plan_record<Work>(plan, a.plan.at_work, record);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int row0 = w.block * SHORT_BLOCK, rows_here = min(SHORT_BLOCK, w.count * G - row0);
  const int row = row0 + min(c, rows_here - 1), m = row / G;  // this lane's query row, its token of the sequence
  const int m_first = row0 / G, m_last = (row0 + rows_here - 1) / G;
  Op q[2];
  query_ops(static_cast<const uint16_t*>(a.q) + (int64_t)(h * G + row - m * G) * a.q_head_stride + (int64_t)(w.token0 + m) * a.q_tok_stride,
            c < rows_here, g, q);
  Running r;
  r.m = -INFINITY, r.l = r.offset = 0.f;
  const float q_sum = query_sum(q);
  for (int db = 0; db < 4; ++db) r.o[db] = f32x4{0, 0, 0, 0};
  const float scale2 = a.scale * LOG2E;
  for (int i = w.u0 + wave; i < w.u1; i += 4) {
    Unit u;
    int rows;
    bool mixed = false;
    if (i < w.n_pages) {
      const Page pg = plan_record<Page>(plan, a.plan.at_pages, w.first_page + i);
      u.bits = page_bits(pg.page);
      u.k = static_cast<const uint8_t*>(a.arena) + page_at(pg.page, a.layer, a.plan.layers, H, h);
      u.v = u.k + (int64_t)H * page_sub(u.bits);
      u.k_stride = u.v_stride = 8 * u.bits;
      u.rows = u.high = rows = pg.rows;
    } else {
      const int first = (i - w.n_pages) * TILE;
      u.bits = 16;
      u.k = static_cast<const uint8_t*>(a.k_new) + 2 * (h * a.kn_head_stride + (int64_t)(w.token0 + first) * a.kn_tok_stride);
      u.v = static_cast<const uint8_t*>(a.v_new) + 2 * (h * a.vn_head_stride + (int64_t)(w.token0 + first) * a.vn_tok_stride);
      u.k_stride = (uint32_t)(2 * a.kn_tok_stride);  // (of a single row, whatever it is)
      u.v_stride = (uint32_t)(2 * a.vn_tok_stride);
      u.rows = min(TILE, w.count - first);
      u.high = min(TILE, m + 1 - first);
      rows = min(TILE, m_last + 1 - first);
      mixed = m_first + 1 - first < rows;
    }
    const int bits = __builtin_amdgcn_readfirstlane(u.bits);
    float* lds = reinterpret_cast<float*>(&o[wave][0][0]);
    if (bits == 4) attend_unit<4, PREC, TERMS>(u, rows, mixed, q, q_sum, scale2, c, g, lds, r);
    else if (bits == 8) attend_unit<8, PREC, TERMS>(u, rows, mixed, q, q_sum, scale2, c, g, lds, r);
    else attend_unit<16, PREC, TERMS>(u, rows, mixed, q, q_sum, scale2, c, g, lds, r);
  }
  r.l = row_sum(r.l);
  r.offset = PREC == 1 ? row_sum(r.offset) : 0.f;
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
  f32x4 x = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float f = __builtin_amdgcn_exp2f(ml[k][rr][0] - ref);
    l += f * ml[k][rr][1];
    x += f * o[k][rr][e4];
  }
  if (w.part < 0) {
    const int at = row0 + rr, tok = at / G;
    store4(a.out, a.out_dtype, (int64_t)(w.token0 + tok) * a.out_tok_stride + (int64_t)(h * G + at - tok * G) * a.out_head_stride + 4 * e4,
           x / l);
  } else {
    const int64_t at = (int64_t)(w.part + rr) * H + h;
    *reinterpret_cast<f32x4*>(part_o + at * D + 4 * e4) = x;
    if (e4 == 0) part_ml[at] = make_float2(top, l);
  }
}

// Joins the partials of 16 query rows: 16 lanes a row, four elements a lane.
__global__ __launch_bounds__(256) void merge_kernel(dkv_paged_args a, const float* part_o, const float2* part_ml) {
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  const int H = a.plan.heads, G = a.plan.q_heads / H, record = blockIdx.x / H, h = blockIdx.x % H;
  if (a.bounds && record >= plan[N_MERGES]) return;
  const Merge w = plan_record<Merge>(plan, a.plan.at_merges, record);
  const int row = w.row0 + (threadIdx.x >> 4), e4 = threadIdx.x & 15;
  if (row >= w.rows) return;
  const int own = w.splits & 0xffff, n = own + (w.splits >> 16);
  auto at = [&](int s) {
    return ((int64_t)(row - w.row0) + (s < own ? w.part + s * w.stride : w.shared + (s - own) * w.shared_stride)) * H + h;
  };
  float top = -INFINITY;
  for (int i = e4; i < n; i += 16) top = fmaxf(top, part_ml[at(i)].x);
#pragma unroll
  for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 16));
  const float ref = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  f32x4 x = {0, 0, 0, 0};
  constexpr int AHEAD = 8;  // splits in flight
  for (int i0 = 0; i0 < n; i0 += AHEAD) {
    float2 p[AHEAD];
    f32x4 o[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t i = at(min(i0 + j, n - 1));
      p[j] = part_ml[i];
      o[j] = *reinterpret_cast<const f32x4*>(part_o + i * D + 4 * e4);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float f = i0 + j < n ? __builtin_amdgcn_exp2f(p[j].x - ref) : 0.f;
      if (i0 + j < n) l += f * p[j].y, x += f * o[j];
    }
  }
  const int tok = row / G;
  store4(a.out, a.out_dtype, (int64_t)(w.token0 + tok) * a.out_tok_stride + (int64_t)(h * G + row - tok * G) * a.out_head_stride + 4 * e4,
         x / l);
}

static int64_t up256(int64_t x) { return (x + 255) & ~(int64_t)255; }

}  // namespace paged
}  // namespace dkv

using namespace dkv;
using namespace dkv::paged;

extern "C" {

int64_t dkv_paged_workspace_bytes(const dkv_paged_args* args) {
  if (!args || args->plan.heads <= 0) return 0;
  const int64_t rows = (int64_t)(args->bounds ? args->plan.max_rows : args->plan.rows) * args->plan.heads;
  return rows > 0 ? up256(4 * D * rows) + up256(8 * rows) : 0;
}

int dkv_paged_attend(const dkv_paged_args* args, void* stream) {
  clear_error();
  if (!args) {
    set_error("dkv_paged_attend: null args");
    return DKV_EINVAL;
  }
  const dkv_paged_args& a = *args;
  if (int rc = check_args(a, true, "dkv_paged_attend")) return rc;
  const int64_t need = dkv_paged_workspace_bytes(args);
  if (need > 0 && (!a.workspace || ((uintptr_t)a.workspace & 15) || a.workspace_bytes < need)) {
    set_error("dkv_paged_attend: workspace of %lld bytes needed, %lld given", (long long)need, (long long)a.workspace_bytes);
    return DKV_EINVAL;
  }
  const hipStream_t st = (hipStream_t)stream;
  const dkv_paged_plan& p = a.plan;
  const int64_t rows = (int64_t)(a.bounds ? p.max_rows : p.rows) * p.heads;
  float* part_o = static_cast<float*>(a.workspace);
  float2* part_ml = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + up256(4 * D * rows));
  const int work = a.bounds ? p.max_work : p.work, merges = a.bounds ? p.max_merges : p.merges;
  const auto attend = a.precision == 1 ? (a.out_dtype == 1 ? short_kernel<1, 3> : short_kernel<1, 2>)
                                       : (a.out_dtype == 1 ? short_kernel<0, 3> : short_kernel<0, 2>);
  if (const int n = a.bounds ? p.max_long : p.long_work) launch_long(a, n, part_o, part_ml, st);
  if (work > 0) hipLaunchKernelGGL(attend, dim3(p.heads * work), dim3(256), 0, st, a, part_o, part_ml);
  if (merges > 0) hipLaunchKernelGGL(merge_kernel, dim3(p.heads * merges), dim3(256), 0, st, a, part_o, part_ml);
  return (int)hipGetLastError();
}

}  // extern "C"
