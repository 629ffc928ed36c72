// Attention of a step's new tokens over pages: the launches, that of few query rows (dkv_paged_short.h) and the join of partial rows
// (gfx950).
#include "dkv_paged_short.h"

namespace dkv {
namespace paged {

using rows::f32x4;

template <int PREC, int TERMS>
__global__ __launch_bounds__(256, 4) void short_kernel(dkv_paged_args a, float* part_o, float2* part_ml) {
  __shared__ __attribute__((aligned(16))) few::ShortShared lds;
  few::short_rows<PREC, TERMS>(a, part_o, part_ml, blockIdx.x, lds);
}

// Joins the partials of 16 query rows: o = sum_s exp(m_s - m) o_s / sum_s exp(m_s - m) l_s. A wave a row, 16 lanes a split with
// four elements each, four splits at a time and AHEAD of these in flight: 4 to 7 us, a launch and its chain of loads. (16 lanes a
// row: 48 branches, whose 127 pages in common were split 64 ways, 13.9 us.)
__global__ __launch_bounds__(256) void merge_kernel(dkv_paged_args a, const float* part_o, const float2* part_ml) {
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  const int H = a.plan.heads, G = a.plan.q_heads / H, h = blockIdx.x % H, four = blockIdx.x / H, record = four / (SHORT_BLOCK / 4);
  if (a.bounds && record >= plan[N_MERGES]) return;
  const Merge w = plan_record<Merge>(plan, a.plan.at_merges, record);
  const int lane = threadIdx.x & 63, e4 = lane & 15, s0 = lane >> 4;
  const int row = w.row0 + four % (SHORT_BLOCK / 4) * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (row >= w.rows) return;
  const int own = w.splits & 0xffff, n = own + (w.splits >> 16);
  auto at = [&](int s) {
    return ((int64_t)(row - w.row0) + (s < own ? w.part + s * w.stride : w.shared + (s - own) * w.shared_stride)) * H + h;
  };
  float top = -INFINITY, l = 0.f;
  f32x4 x = {0, 0, 0, 0};
  constexpr int AHEAD = 5;  // (a token of 48 branches / of 64 streams / 16 questions: 4 18.3 / 31.7 / 33.7 us, 5 17.8 / 31.4 / 33.6, 8 18.5 / 32.2 / 35.7)
  for (int i0 = 0; i0 < n; i0 += 4 * AHEAD) {
    float2 p[AHEAD];
    f32x4 o[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t i = at(min(i0 + 4 * j + s0, n - 1));
      p[j] = part_ml[i];
      o[j] = *reinterpret_cast<const f32x4*>(part_o + i * D + 4 * e4);
    }
    float here = top;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i0 + 4 * j + s0 >= n) p[j] = make_float2(-INFINITY, 0.f), o[j] = f32x4{0, 0, 0, 0};
      here = fmaxf(here, p[j].x);
    }
    const float ref = here == -INFINITY ? 0.f : here, alpha = __builtin_amdgcn_exp2f(top - ref);
    l *= alpha, x *= alpha;
    top = here;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float f = __builtin_amdgcn_exp2f(p[j].x - ref);
      l += f * p[j].y;
      x += f * o[j];
    }
  }
  const float all = rows::row_max(top), ref = all == -INFINITY ? 0.f : all, f = __builtin_amdgcn_exp2f(top - ref);
  l = rows::row_sum(l * f);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = rows::row_sum(x[e] * f);
  const int tok = row / G;
  if (s0 == 0)
    store4(a.out, a.out_dtype, (int64_t)(w.token0 + tok) * a.out_tok_stride + (int64_t)(h * G + row - tok * G) * a.out_head_stride + 4 * e4,
           x / l);
}

// Up to so many units of few query rows a CU (over all heads) go behind the workgroups of many in one launch, which has half as many
// waves for them. One launch / two, us: 16 questions, 260 workgroups, 33.5 / 40.6; a prompt of 200 tokens beside a token of each of 8
// sequences of 2000 tokens (6 units a CU) 14.4 / 21.3, 24 of 8000 (60) 43.7 / 48.1, 64 of 2000 (41) 35.0 / 39.3 and at precision 1
// 36.7 / 42.6, 64 of 8000 (160) 86 / 82, 6 of 100k (185) 101 / 94.
constexpr int64_t TOGETHER = 64, CUS = 256;

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
  // (At precision 1 a weight meets codes whose offset comes apart: two terms would be off by 2^-18 of a row's range.)
  const auto attend = a.precision == 1 ? short_kernel<1, 3> : a.out_dtype == 1 ? short_kernel<0, 3> : short_kernel<0, 2>;
  const int n_long = a.bounds ? p.max_long : p.long_work;
  const bool together = n_long > 0 && !a.bounds && (int64_t)p.units * p.heads <= TOGETHER * CUS;
  if (n_long > 0) launch_long(a, n_long, together ? work : 0, part_o, part_ml, st);
  if (work > 0 && !together) hipLaunchKernelGGL(attend, dim3(p.heads * work), dim3(256), 0, st, a, part_o, part_ml);
  if (merges > 0) hipLaunchKernelGGL(merge_kernel, dim3(p.heads * merges * (SHORT_BLOCK / 4)), dim3(256), 0, st, a, part_o, part_ml);
  return (int)hipGetLastError();
}

}  // extern "C"
