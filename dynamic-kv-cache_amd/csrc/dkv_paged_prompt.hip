// Prompts over pages (gfx950): sequences (and groups that share pages) of many query rows.
//
// A workgroup of 8 waves takes LONG_BLOCK query rows of a KV head, 32 a wave, over a range of units of 64 keys, and
// brings every unit's K and V to LDS once for all of them: packed rows through registers, where they are unpacked, new
// rows straight (global_load_lds). S^T = K Q^T and O^T = V^T P^T as v_mfma_f32_32x32x16_bf16 with keys on M of the
// first product and query rows on N of both, so lane l holds the scores of query row l % 32 (keys 8 a + 4 (l / 32) + i)
// in the places that the second product reads P^T from: P never leaves its registers, and a row's maximum and sum take
// one exchange between the two halves of a wave. V^T comes from V's rows in LDS by transposing reads (ds_read_b64_tr_b16:
// of 16 lanes that read 4 elements of 4 rows each, lane i gets element i of the rows).
#include "dkv_rows.h"
#include "dkv_paged.h"

namespace dkv {
namespace paged {

using rows::bf16x8;
using rows::CENTRE;
using rows::split_pair;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

union Op8 {
  bf16x8 v;
  u32x4 u;
  s16x4 h[2];
};

constexpr int WAVES = LONG_BLOCK / 32;
constexpr int RING = 3;          // units in LDS: one is read, one arrives, one is written
constexpr int TILE_BYTES = 8192;  // K or V of a unit: row r's 16-byte piece p lies at r * 128 + (p ^ r % 8) * 16

// A unit that comes through registers: a page's rows, or new ones that not all of the workgroup's query rows see.
struct Source {
  const uint8_t* k;
  const uint8_t* v;
  uint32_t k_stride, v_stride;  // bytes from row to row
  int bits, rows;               // rows that are there
  bool page;
};

struct Raw {  // a thread's 8 elements of a row of K and of V
  u32x4 k, v;
  float2 ka, va;
};

// 8 elements of a packed row as bf16: their values (PREC 0), or the centred codes, whose scale and offset come later.
template <int PREC>
__device__ __forceinline__ u32x4 unpack8(int bits, const u32x4& w, const float2& as) {
  if (bits == 16) return w;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)(bits == 4 ? (w[0] >> (4 * e)) & 15u : (w[e >> 2] >> (8 * (e & 3))) & 255u);
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = bits == 4 ? CENTRE<4> : CENTRE<8>;
    out[i] = PREC ? pack_bf16(x[2 * i] - c, x[2 * i + 1] - c) : pack_bf16(x[2 * i] * as.y + as.x, x[2 * i + 1] * as.y + as.x);
  }
  return out;
}

// max(a, b, c) of values that are never NaN (see max_nn).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

template <int PREC, int TERMS>
__global__ __launch_bounds__(64 * WAVES, PREC ? 2 : 4) void long_kernel(dkv_paged_args a, float* part_o, float2* part_ml) {
  __shared__ __attribute__((aligned(1024))) uint8_t tiles[RING][2][TILE_BYTES];
  __shared__ int bad;  // a new value that is infinite or NaN was taken for zero
  __shared__ __attribute__((aligned(16))) float2 scales[PREC ? RING : 1][2][PREC ? TILE : 1];  // {offset + scale * centre, scale}
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  const int H = a.plan.heads, G = a.plan.q_heads / H, record = blockIdx.x / H, h = blockIdx.x % H;
  if (a.bounds && record >= plan[N_LONG]) return;
  const Work w = plan_record<Work>(plan, a.plan.at_long, record);
  auto page = [&](int u) { return plan_record<Page>(plan, a.plan.at_pages, w.first_page + u); };
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, c = lane & 31, half = lane >> 5;
  const int total = w.count * G, wave0 = w.block * LONG_BLOCK + 32 * wave;  // the wave's first query row
  const bool on = wave0 < total;
  const int row = min(wave0 + c, total - 1), m = row / G;  // this lane's query row and its token
  const int m_first = min(wave0, total - 1) / G, m_last = min(wave0 + 31, total - 1) / G;
  const int srow = t >> 3, piece = (t & 7) ^ (srow & 7);  // of the tiles' rows, this thread's 8 elements 8 * piece

  // Units from here on come straight to LDS while every query row of the workgroup sees all of their keys.
  const int seen_by_all = w.n_pages + (min(w.block * LONG_BLOCK, total - 1) / G + 1) / TILE;
  auto straight = [&](int u) { return u >= w.n_pages && u < seen_by_all; };
  auto source = [&](int u) {
    Source s;
    s.page = u < w.n_pages;
    if (s.page) {
      const Page p = page(u);
      s.bits = page_bits(p.page), s.rows = p.rows;
      s.k = static_cast<const uint8_t*>(a.arena) + page_at(p.page, a.layer, a.plan.layers, H, h);
      s.v = s.k + (int64_t)H * page_sub(s.bits);
      s.k_stride = s.v_stride = 8 * s.bits;
    } else {
      const int first = (u - w.n_pages) * TILE;
      s.bits = 16, s.rows = min(TILE, w.count - first);
      s.k = static_cast<const uint8_t*>(a.k_new) + 2 * (h * a.kn_head_stride + (int64_t)(w.token0 + first) * a.kn_tok_stride);
      s.v = static_cast<const uint8_t*>(a.v_new) + 2 * (h * a.vn_head_stride + (int64_t)(w.token0 + first) * a.vn_tok_stride);
      s.k_stride = (uint32_t)(2 * a.kn_tok_stride), s.v_stride = (uint32_t)(2 * a.vn_tok_stride);
    }
    return s;
  };
  auto load_raw = [&](const Source& s, Raw& r) {
    const int at = srow < s.rows ? srow : 0;
    const uint8_t* k = s.k + (__umul24(at, s.k_stride) + s.bits * piece);
    const uint8_t* v = s.v + (__umul24(at, s.v_stride) + s.bits * piece);
    if (s.bits == 4) {
      r.k[0] = *reinterpret_cast<const uint32_t*>(k);
      r.v[0] = *reinterpret_cast<const uint32_t*>(v);
    } else if (s.bits == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(k), y = *reinterpret_cast<const uint2*>(v);
      r.k[0] = x.x, r.k[1] = x.y, r.v[0] = y.x, r.v[1] = y.y;
    } else {
      r.k = *reinterpret_cast<const u32x4*>(k);
      r.v = *reinterpret_cast<const u32x4*>(v);
    }
    if (s.bits < 16) {
      r.ka = *reinterpret_cast<const float2*>(s.k + TILE * 8 * s.bits + 8 * at);
      r.va = *reinterpret_cast<const float2*>(s.v + TILE * 8 * s.bits + 8 * at);
    }
  };
  auto write_raw = [&](const Source& s, const Raw& r, int buf) {
    const bool there = srow < s.rows;  // (rows that are not there: zeros, which meet a p of zero)
    const u32x4 k = unpack8<PREC>(s.bits, r.k, r.ka);
    u32x4 v = unpack8<PREC>(s.bits, r.v, r.va);
    if (!s.page) {  // an infinite or NaN value meets a p of zero where it is not seen: zero, and added after all units
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t keep = (bad_bf16(v[e]) ? 0u : 0xffffu) | (bad_bf16(v[e] >> 16) ? 0u : 0xffff0000u);
        if (there && keep != 0xffffffffu) bad = 1;
        v[e] &= keep;
      }
    }
    *reinterpret_cast<u32x4*>(&tiles[buf][0][16 * t]) = there ? k : u32x4{0, 0, 0, 0};
    *reinterpret_cast<u32x4*>(&tiles[buf][1][16 * t]) = there ? v : u32x4{0, 0, 0, 0};
    if (PREC && (t & 7) == 0) {
      const float centre = s.bits == 4 ? CENTRE<4> : CENTRE<8>;
      const bool scaled = there && s.bits < 16;
      scales[buf][0][srow] = scaled ? make_float2(__builtin_fmaf(r.ka.y, centre, r.ka.x), r.ka.y) : make_float2(0.f, 1.f);
      scales[buf][1][srow] = scaled ? make_float2(__builtin_fmaf(r.va.y, centre, r.va.x), r.va.y) : make_float2(0.f, there ? 1.f : 0.f);
    }
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&tiles[0][0][0];
  auto load_new = [&](int u, int buf) {  // 64 new tokens, all there
    const int tok = w.token0 + (u - w.n_pages) * TILE + srow;
    const uint32_t to = lds0 + buf * (2 * TILE_BYTES) + 1024 * wave;
    load_piece(static_cast<const uint16_t*>(a.k_new) + h * a.kn_head_stride + tok * a.kn_tok_stride + 8 * piece, to);
    load_piece(static_cast<const uint16_t*>(a.v_new) + h * a.vn_head_stride + tok * a.vn_tok_stride + 8 * piece, to + TILE_BYTES);
  };

  Op8 q[4];
  {
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(h * G + row - m * G) * a.q_head_stride +
                          (int64_t)(w.token0 + m) * a.q_tok_stride + 8 * half;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) q[ks].u = *reinterpret_cast<const u32x4*>(src + 16 * ks);
  }
  Raw raw;
  Source ahead{};  // the unit in `raw`
  if (t == 0) bad = 0;
  __syncthreads();
  // the first unit to LDS, the second on its way
  if (w.u0 < w.u1) {
    if (straight(w.u0)) {
      load_new(w.u0, 0);
    } else {
      ahead = source(w.u0);
      load_raw(ahead, raw);
      write_raw(ahead, raw, 0);
    }
    if (w.u0 + 1 < w.u1) {
      if (straight(w.u0 + 1)) {
        load_new(w.u0 + 1, 1);
      } else {
        ahead = source(w.u0 + 1);
        load_raw(ahead, raw);
      }
    }
  }
  float q_sum = 0.f;  // of the query row's elements
  if (PREC) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int j = 0; j < 4; ++j) q_sum += bf16_lo(q[ks].u[j]) + bf16_hi(q[ks].u[j]);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(q_sum), __float_as_uint(q_sum), false, false);
    q_sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  f32x16 acc[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[0][i] = acc[1][i] = 0.f;
  float m_run = -INFINITY, l_part = 0.f, offset = 0.f;  // (l_part and offset: of this lane's keys)
  const float xs = a.scale * LOG2E;
  // This lane's LDS places: pieces of key c for the K operands, and the 4 elements it reads for the V^T operands.
  // (Piece 2 ks + half of a row lies 32 ks further on but for the carry, the same bits in the other order: ^.)
  const uint32_t k_at = c * 128 + ((half ^ (c & 7)) << 4);
  uint32_t v_at;
  {
    const int i = lane & 15, vr = 4 * half + (i >> 2), sub = (lane >> 4) & 1;
    v_at = vr * 128 + (((2 * sub + ((i & 3) >> 1)) ^ (vr & 7)) << 4) + 8 * (i & 1);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();

  int buf = 0;
  for (int u = w.u0; u < w.u1; ++u) {
    const int next = buf + 1 == RING ? 0 : buf + 1, after = next + 1 == RING ? 0 : next + 1;
    int rows_here = TILE;
    if (u < w.n_pages) rows_here = page(u).rows;
    const bool packed = PREC && u < w.n_pages;
    if (u + 1 < w.u1 && !straight(u + 1)) write_raw(ahead, raw, next);
    bool direct = false;  // rows were asked for straight to LDS in this iteration
    if (u + 2 < w.u1) {
      if (straight(u + 2)) {
        load_new(u + 2, after);
        direct = true;
      } else {
        ahead = source(u + 2);
        load_raw(ahead, raw);
      }
    }
    const int first = (u - w.n_pages) * TILE;
    if (on && (u < w.n_pages || first <= m_last)) {
      const uint8_t* kt = &tiles[buf][0][0];
      const uint8_t* vt = &tiles[buf][1][0];
      const int high = u < w.n_pages ? rows_here : m + 1 - first;  // keys below are visible to this lane's row
      const bool masked = u < w.n_pages ? rows_here < TILE : first + TILE - 1 > m_first;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {  // 32 keys at a time
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          Op8 k;
          k.u = *reinterpret_cast<const u32x4*>(kt + (k_at ^ (32 * ks)) + 4096 * kb);
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k.v, q[ks].v, s, 0, 0, 0);
        }
        // max3 below is a statement of its own, before which the compiler does not wait for a matrix product's result: 19
        // states after one of 16 passes.
        asm volatile("s_nop 15\n s_nop 7" : "+v"(s));
        if (packed) {
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const f32x4 as = *reinterpret_cast<const f32x4*>(&scales[buf][0][32 * kb + 8 * (i / 4) + 4 * half + i % 4]);
            s[i] = __builtin_fmaf(as[1], s[i], as[0] * q_sum);
            s[i + 1] = __builtin_fmaf(as[3], s[i + 1], as[2] * q_sum);
          }
        }
        if (masked)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = 32 * kb + 8 * (i / 4) + 4 * half + i % 4 < high ? s[i] : -INFINITY;
        float top = max3(s[0], s[1], s[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) top = max3(top, s[i], s[i + 1]);
        top = max_nn(top, s[15]);
        // The running maximum moves when some lane's scores pass it; only then do a row's two lanes exchange theirs.
        if (__builtin_amdgcn_ballot_w64(top * xs > m_run)) {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
          const float mnew = max_nn(m_run, max_nn(__uint_as_float(x[0]), __uint_as_float(x[1])) * xs);
          const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - mnew);
          m_run = mnew;
          l_part *= alpha;
          if (PREC) offset *= alpha;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[0][i] *= alpha, acc[1][i] *= alpha;
        }
        const float mref = m_run == -INFINITY ? 0.f : m_run;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], xs, -mref));
          sum += s[i];
        }
        l_part += sum;
#pragma unroll
        for (int st = 0; st < 2; ++st) {  // 16 keys
          Op8 p[TERMS];
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            float p0 = s[8 * st + j], p1 = s[8 * st + j + 1];
            if (packed) {
              const f32x4 as = *reinterpret_cast<const f32x4*>(&scales[buf][1][32 * kb + 16 * st + 8 * (j / 4) + 4 * half + j % 4]);
              offset = __builtin_fmaf(p0, as[0], offset);
              offset = __builtin_fmaf(p1, as[2], offset);
              p0 *= as[1], p1 *= as[3];
            }
            uint32_t x[TERMS];
            split_pair<TERMS>(p0, p1, x);
#pragma unroll
            for (int k = 0; k < TERMS; ++k) p[k].u[j / 2] = x[k];
          }
#pragma unroll
          for (int db = 0; db < 2; ++db) {
            Op8 v;
#pragma unroll
            for (int j = 0; j < 2; ++j)
              v.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) s16x4*)(vt + (v_at ^ (64 * db)) + (32 * kb + 16 * st + 8 * j) * 128));
#pragma unroll
            for (int k = TERMS - 1; k >= 0; --k) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v.v, p[k].v, acc[db], 0, 0, 0);
          }
        }
      }
    }
    // The next unit has landed (its direct loads were issued an iteration ago: at most this one's two are under way)
    // and is written, by every wave, and no wave reads this one any more.
    if (direct) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    else if (straight(u + 1)) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    buf = next;
  }
  if (!on) return;
  auto both = [](float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
  };
  const float l = both(l_part), off = PREC ? both(offset) : 0.f;
  if (bad) {  // (rare) new values that the products took for zero, with their weights computed again
    for (int u = max(w.u0, seen_by_all); u < w.u1; ++u) {
      const int first = (u - w.n_pages) * TILE;
      for (int j = 0; j < min(TILE, w.count - first); ++j) {
        const int64_t tok = w.token0 + first + j;
        const uint2* v = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.v_new) + h * a.vn_head_stride + tok * a.vn_tok_stride);
        uint2 x[8];
        bool some = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // elements 8 i + 4 half + ...
          x[i] = v[2 * i + half];
          some = some || bad_bf16(x[i].x) || bad_bf16(x[i].x >> 16) || bad_bf16(x[i].y) || bad_bf16(x[i].y >> 16);
        }
        if (!__builtin_amdgcn_ballot_w64(some)) continue;
        const u32x4* k = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.k_new) + h * a.kn_head_stride + tok * a.kn_tok_stride);
        float dot = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const u32x4 y = k[2 * ks + half];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dot = __builtin_fmaf(bf16_lo(q[ks].u[e]), bf16_lo(y[e]), __builtin_fmaf(bf16_hi(q[ks].u[e]), bf16_hi(y[e]), dot));
        }
        const float p = __builtin_amdgcn_exp2f(both(dot) * xs - m_run);
        if (first + j > m) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int db = i / 4, at = 4 * (i % 4);
          if (bad_bf16(x[i].x)) acc[db][at] += p * bf16_lo(x[i].x);
          if (bad_bf16(x[i].x >> 16)) acc[db][at + 1] += p * bf16_hi(x[i].x);
          if (bad_bf16(x[i].y)) acc[db][at + 2] += p * bf16_lo(x[i].y);
          if (bad_bf16(x[i].y >> 16)) acc[db][at + 3] += p * bf16_hi(x[i].y);
        }
      }
    }
  }
  if (wave0 + c >= total) return;
  if (w.part < 0) {
    const float inv = 1.f / l;
    const int64_t at = (int64_t)(w.token0 + m) * a.out_tok_stride + (int64_t)(h * G + row - m * G) * a.out_head_stride + 4 * half;
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const f32x4 x = f32x4{acc[i / 16][i % 16] + off, acc[i / 16][i % 16 + 1] + off, acc[i / 16][i % 16 + 2] + off, acc[i / 16][i % 16 + 3] + off} * inv;
      store4(a.out, a.out_dtype, at + 32 * (i / 16) + 8 * (i % 16 / 4), x);
    }
  } else {
    const int64_t at = (int64_t)(w.part + 32 * wave + c) * H + h;
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<f32x4*>(part_o + at * D + 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * half) =
          f32x4{acc[i / 16][i % 16] + off, acc[i / 16][i % 16 + 1] + off, acc[i / 16][i % 16 + 2] + off, acc[i / 16][i % 16 + 3] + off};
    if (half == 0) part_ml[at] = make_float2(m_run, l);
  }
}

void launch_long(const dkv_paged_args& a, int work, float* part_o, float2* part_ml, hipStream_t s) {
  const auto kernel = a.precision == 1 ? (a.out_dtype == 1 ? long_kernel<1, 3> : long_kernel<1, 2>)
                                       : (a.out_dtype == 1 ? long_kernel<0, 3> : long_kernel<0, 1>);
  hipLaunchKernelGGL(kernel, dim3(work * a.plan.heads), dim3(64 * WAVES), 0, s, a, part_o, part_ml);
}

}  // namespace paged
}  // namespace dkv
