// Prompts over pages (gfx950): sequences (and groups that share pages) of many query rows.
//
// A workgroup of 8 waves takes LONG_BLOCK query rows of a KV head, 32 a wave, over a range of units of 64 keys, and
// brings every unit's K and V to LDS once for all of them: packed rows through registers, where they are unpacked, new
// rows straight (global_load_lds). S^T = K Q^T and O^T = V^T P^T as v_mfma_f32_32x32x16_bf16 with keys on M of the
// first product and query rows on N of both, so lane l holds the scores of query row l % 32 (keys 8 a + 4 (l / 32) + i)
// in the places that the second product reads P^T from: P never leaves its registers, and a row's maximum and sum take
// one exchange between the two halves of a wave. V^T comes from V's rows in LDS by transposing reads (ds_read_b64_tr_b16:
// of 16 lanes that read 4 elements of 4 rows each, lane i gets element i of the rows).
//
// Packed rows of unit u + 3 are asked for, and those of u + 1 unpacked, while u is multiplied; new and 16-bit rows come two units
// ahead; one barrier a unit. Scores, statistics and sums are fp32. P is one bf16 value at precision and output bf16 (a relative 2^-8
// of each weight, averaged over the keys; a sequence of few rows keeps two, dkv_paged_short.h), else the sum of three
// (at precision fp32 for either output: a weight meets a code that is up to half a row's range from its offset, whatever is left of
// the two).
// What bounds it: the vector units, some 180 instructions a unit and wave beside its 16 matrix products of 32 cycles, of them 32
// exponentials of twice the cost or more: 12.5k tokens of prompts of 5 heads of 3 209 us (791 TFLOP/s, 60 % of a large product's; vector units busy 62 % of the time, matrix units 35), 12
// prompts of up to 2048 tokens of 8 heads of 4 56 us (615); with few units a workgroup the chain from the plan to the first tile, 16
// questions about 6144 shared tokens 27 us. At fp32 the split into three values and the scales apart, some 500 instructions a unit
// and wave: 8 frames of 78 tokens over 92k 71 us (62 and 23 %).

#include <type_traits>

#include "dkv_paged_short.h"

namespace dkv {
namespace paged {

using rows::bf16x8;
using rows::CENTRE;
using rows::split_pair;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

union Op8 {
  bf16x8 v;
  u32x4 u;
  s16x4 h[2];
};

constexpr int WAVES = LONG_BLOCK / 32;
constexpr int RING = 3;           // units' tiles in LDS (one is read, one is written or has arrived, one arrives), and packed units
constexpr int TILE_BYTES = 8192;  // K or V of a unit: row r's 16-byte piece p lies at r * 128 + (p ^ place(r)) * 16
constexpr int RAW_V = 4096, RAW_SCALES = 8192, RAW_BYTES = 9216;  // a packed unit as it is stored: K, V, (offset, scale) of K and V

// Rows of equal parity share banks. This order keeps apart the equal pieces of rows {0-3, 12-15, 20-23, 24-27} (and these
// + 4, + 8, + 16), which one step of a 16-byte read takes, and the four neighbouring pieces of rows 4 n + {0, 2}, which the
// transposing reads do.
__device__ __forceinline__ int place(int row) { return (row >> 1 & 1) << 2 | (row >> 3 & 1) << 1 | (row >> 2 & 1); }

// load_piece (dkv_common.h) from an address that a wave shares and an offset of each lane.
__device__ __forceinline__ void load_piece_at(const uint8_t* from, uint32_t offset, uint32_t to) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n s_mov_b32 m0, %3\n s_nop 0\n global_load_lds_dwordx4 %1, %2\n s_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(offset), "s"(from), "s"(to) : "memory");
}

// 8 elements of a packed row as bf16: their values (PREC 0), or the centred codes, whose scale and offset come later.
template <int PREC>
__device__ __forceinline__ u32x4 unpack8(int bits, const uint2& w, const float2& as) {
  float x[8];
  const uint32_t even = bits == 4 ? w.x & 0x0f0f0f0fu : w.x, odd = bits == 4 ? (w.x >> 4) & 0x0f0f0f0fu : w.y;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (float)((even >> (8 * e)) & 255u), x[4 + e] = (float)((odd >> (8 * e)) & 255u);
  const float c = bits == 4 ? CENTRE<4> : CENTRE<8>;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = PREC ? x[e] - c : x[e] * as.y + as.x;
  if (bits == 4)  // (bytes of `even` and `odd` are every other element)
    return u32x4{pack_bf16(x[0], x[4]), pack_bf16(x[1], x[5]), pack_bf16(x[2], x[6]), pack_bf16(x[3], x[7])};
  return u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

// At most n loads straight to LDS of this wave are under way.
__device__ __forceinline__ void wait_loads(int n) {
  if (n == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else if (n == 1) asm volatile("s_waitcnt vmcnt(1)" ::: "memory");
  else if (n == 2) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(3)" ::: "memory");
}

// max(a, b, c) of values that are never NaN (see max_nn).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// x as a value of its own: what is computed from it is not kept in registers from before. (These are full: addresses that are used
// once a unit or less would be kept in scratch memory.)
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Workgroups behind the first n_long records' take those of few query rows, in the first half of their threads.
template <int PREC, int TERMS, int FEW_TERMS>
__global__ __launch_bounds__(64 * WAVES, 4) void long_kernel(dkv_paged_args a, int n_long, float* part_o, float2* part_ml) {
  __shared__ __attribute__((aligned(1024))) uint8_t tiles[RING][2][TILE_BYTES];
  __shared__ __attribute__((aligned(1024))) uint8_t packed_rows[RING][RAW_BYTES];
  __shared__ __attribute__((aligned(16))) float2 scales[PREC ? RING : 1][2][PREC ? TILE : 1];  // {offset + scale * centre, scale}
  __shared__ int bad;  // a new value that is infinite or NaN was taken for zero
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  const int H = a.plan.heads, G = a.plan.q_heads / H, record = blockIdx.x / H, h = blockIdx.x % H;
  if (record >= n_long) {
    static_assert(sizeof(few::ShortShared) <= sizeof(tiles), "in the tiles' place");
    if (threadIdx.x < 256) few::short_rows<PREC, FEW_TERMS>(a, part_o, part_ml, blockIdx.x - n_long * H, *reinterpret_cast<few::ShortShared*>(&tiles[0][0][0]));
    return;
  }
  if (a.bounds && record >= plan[N_LONG]) return;
  const Work w = plan_record<Work>(plan, a.plan.at_long, record);
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, c = lane & 31, half = lane >> 5;
  const int total = w.count * G, wave0 = w.block * LONG_BLOCK + 32 * wave;  // the wave's first query row
  const bool on = wave0 < total;
  const int row = min(wave0 + c, total - 1), m = row / G;  // this lane's query row and its token
  const int first_token = w.block * LONG_BLOCK / G;  // of the workgroup's query rows
  const int m_first = min(wave0, total - 1) / G, m_last = min(wave0 + 31, total - 1) / G;
  const int srow = t >> 3, piece = (t & 7) ^ place(srow);  // of the tiles' rows, this thread's 8 elements 8 * piece

  // A unit: 64 rows (`rows` of them there) of a page or of the new tokens, and how many loads of it this wave issues.
  struct Unit {
    int bits, rows, loads;
    uint32_t page;
  };
  auto unit_at = [&](int u) {
    Unit x{16, 0, 0, 0};
    if (u >= w.u1) return x;
    if (u < w.n_pages) {
      const Page p = plan_record<Page>(plan, a.plan.at_pages, w.first_page + u);
      x.bits = page_bits(p.page), x.rows = p.rows, x.page = p.page;
    } else {
      x.rows = min(TILE, w.count - (u - w.n_pages) * TILE);
    }
    x.loads = x.bits == 16 ? 2 : x.bits == 8 ? 1 + (wave == 0) : (wave & 3) < 2 || wave == 2;
    return x;
  };
  const uint32_t tile0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&tiles[0][0][0];
  const uint32_t raw0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&packed_rows[0][0];
  const uint8_t* const base = static_cast<const uint8_t*>(a.arena);
  const int64_t grain = grain_bytes(a.plan.layers, H), sub = (int64_t)a.layer * 2 * H + h;
  // Rows of 16 bits go straight to their tile: a wave 8 rows of K and of V. New rows past the last one repeat it; rows of a
  // page that are not there are read as they are (zero_values). New rows are attended to without scales.
  auto load_rows = [&](auto of_page, const uint8_t* k, const uint8_t* v, int rows, uint32_t k_stride, uint32_t v_stride, int buf) {
    const int thread = anew(t), srow = thread >> 3, piece = (thread & 7) ^ place(srow), r = min(srow, rows - 1);
    const uint32_t to = tile0 + buf * (2 * TILE_BYTES) + 1024 * wave;
    load_piece_at(k, 16 * piece + __umul24(r, k_stride), to);
    load_piece_at(v, 16 * piece + __umul24(r, v_stride), to + TILE_BYTES);
    if (PREC && of_page && (thread & 7) == 0) scales[buf][0][srow] = scales[buf][1][srow] = make_float2(0.f, 1.f);
  };
  const uint32_t kn_stride = (uint32_t)(2 * a.kn_tok_stride), vn_stride = (uint32_t)(2 * a.vn_tok_stride);  // (of a single row, whatever it is)
  auto new_rows = [&](const void* x, int64_t head_stride, int64_t tok_stride, int u) {
    return static_cast<const uint8_t*>(x) + 2 * (h * head_stride + ((int64_t)w.token0 + (u - w.n_pages) * TILE) * tok_stride);
  };
  auto load_tile = [&](int u, const Unit& x, int buf) {
    if (u < w.n_pages) {
      const uint8_t* k = base + (x.page >> 2) * grain + sub * page_sub(16);
      load_rows(std::true_type(), k, k + (int64_t)H * page_sub(16), TILE, 128, 128, buf);
    } else {
      load_rows(std::false_type(), new_rows(a.k_new, a.kn_head_stride, a.kn_tok_stride, u),
                new_rows(a.v_new, a.vn_head_stride, a.vn_tok_stride, u), x.rows, kn_stride, vn_stride, buf);
    }
  };
  // Packed rows come as they are: at 8 bits a wave 1 KB of K (waves 0 to 3) or V, at 4 bits every other wave, and one wave
  // the (offset, scale) pairs.
  auto load_raw = [&](const Unit& x, int buf) {
    const int lane = anew(t) & 63;
    const uint8_t* k = base + (x.page >> 2) * grain + sub * page_sub(x.bits);
    const uint32_t to = raw0 + buf * RAW_BYTES, kv = H * page_sub(x.bits);  // (a page's V lies that far behind its K)
    if (x.bits == 8 || (wave & 3) < 2)
      load_piece_at(k + (wave < 4 ? 0 : kv) + 1024 * (wave & 3), 16 * lane, to + (wave < 4 ? 0 : RAW_V) + 1024 * (wave & 3));
    if (wave == (x.bits == 8 ? 0 : 2)) load_piece_at(k, TILE * 8 * x.bits + 16 * (lane & 31) + (lane < 32 ? 0 : kv), to + RAW_SCALES);
  };
  auto unpack = [&](const Unit& x, int raw_buf, int buf) {
    const uint8_t* from = packed_rows[raw_buf];
    const float2 ka = reinterpret_cast<const float2*>(from + RAW_SCALES)[srow], va = reinterpret_cast<const float2*>(from + RAW_SCALES)[TILE + srow];
    uint2 k, v;
    if (x.bits == 4) {
      k.x = *reinterpret_cast<const uint32_t*>(from + srow * 32 + 4 * piece);
      v.x = *reinterpret_cast<const uint32_t*>(from + RAW_V + srow * 32 + 4 * piece);
    } else {
      const int at = srow * 64 + 8 * anew(piece);
      k = *reinterpret_cast<const uint2*>(from + at);
      v = *reinterpret_cast<const uint2*>(from + RAW_V + at);
    }
    const bool there = srow < x.rows;  // (rows that are not there: zeros, which meet a p of zero)
    const u32x4 ku = unpack8<PREC>(x.bits, k, ka), vu = unpack8<PREC>(x.bits, v, va);
    *reinterpret_cast<u32x4*>(&tiles[buf][0][16 * t]) = there ? ku : u32x4{0, 0, 0, 0};
    *reinterpret_cast<u32x4*>(&tiles[buf][1][16 * t]) = there ? vu : u32x4{0, 0, 0, 0};
    if (PREC && (t & 7) == 0) {
      const float centre = x.bits == 4 ? CENTRE<4> : CENTRE<8>;
      scales[buf][0][srow] = there ? make_float2(__builtin_fmaf(ka.y, centre, ka.x), ka.y) : make_float2(0.f, 0.f);
      scales[buf][1][srow] = there ? make_float2(__builtin_fmaf(va.y, centre, va.x), va.y) : make_float2(0.f, 0.f);
    }
  };
  // Values of a tile that would make NaN of a weight of zero become zeros: of rows that are not there, and infinite or NaN
  // ones of new rows (added after all units). Each thread looks at its own 16 bytes.
  auto zero_values = [&](const Unit& x, uint8_t* vt, bool fresh) {
    u32x4* at = reinterpret_cast<u32x4*>(vt + 16 * t);
    const bool there = srow < x.rows;
    u32x4 y = *at;
    bool changed = !there;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t keep = !there ? 0u : !fresh ? 0xffffffffu : (bad_bf16(y[e]) ? 0u : 0xffffu) | (bad_bf16(y[e] >> 16) ? 0u : 0xffff0000u);
      changed = changed || keep != 0xffffffffu;
      y[e] &= keep;
    }
    if (changed) *at = y;
    if (changed && there) bad = 1;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  Op8 q[4];
  {
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(h * G + row - m * G) * a.q_head_stride +
                          (int64_t)(w.token0 + m) * a.q_tok_stride + 8 * half;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) q[ks].u = *reinterpret_cast<const u32x4*>(src + 16 * ks);
  }
  if (t == 0) bad = 0;
  // Units u, u + 1, u + 2 and u + 3. Packed ones are asked for three units ahead, unpacked one ahead; the others two ahead.
  Unit x0 = unit_at(w.u0), x1 = unit_at(w.u0 + 1), x2 = unit_at(w.u0 + 2), x3 = unit_at(w.u0 + 3);
  if (x0.bits < 16) load_raw(x0, 0);
  else if (x0.rows) load_tile(w.u0, x0, 0);
  if (x1.bits < 16) load_raw(x1, 1);
  else if (x1.rows) load_tile(w.u0 + 1, x1, 1);
  if (x2.bits < 16) load_raw(x2, 2);
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
  const uint32_t k_at = c * 128 + ((half ^ place(c)) << 4);
  uint32_t v_at;
  {
    const int i = lane & 15, vr = 4 * half + (i >> 2), sub = (lane >> 4) & 1;
    v_at = vr * 128 + (((2 * sub + ((i & 3) >> 1)) ^ place(vr)) << 4) + 8 * (i & 1);
  }
  // (The query operands have arrived: a wait for them inside the loop would drain the loads under way in every iteration.)
  asm volatile("" ::"v"(q[0].u), "v"(q[1].u), "v"(q[2].u), "v"(q[3].u));
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (x0.bits < 16) {
    unpack(x0, 0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // A unit's keys from its tiles; SCALED: their scales and offsets are to come (PREC 1, pages; those of 16-bit ones are 1 and 0: a
  // path of their own in that loop takes 221 registers, one workgroup a CU, 8 frames 101 us instead of 77; new tokens' loop has one,
  // 15 prompts of 645 tokens 97 us, 108 without). Keys from `high` on are not visible to this lane's
  // row, none from 32 on to any row of the wave where there is one half.
  auto attend = [&](auto scaled, int buf, bool masked, int high, bool one_half) {
    constexpr bool SCALED = decltype(scaled)::value;
    constexpr int AHEAD = 4;  // operands of K under way (12.5k tokens of prompts 2: 224.4 us, 4: 223.5, 6: 225.2)
    const uint8_t* kt = &tiles[buf][0][0];
    const uint8_t* vt = &tiles[buf][1][0];
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
    __builtin_amdgcn_s_setprio(1);  // (products before the other waves' exponentials: 0.7 %)
    Op8 k[AHEAD];
    auto load_k = [&](int i) { k[i % AHEAD].u = *reinterpret_cast<const u32x4*>(kt + (k_at ^ (32 * (i / 2))) + 4096 * (i % 2)); };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load_k(i);
    __builtin_amdgcn_sched_barrier(0);  // (the compiler would read each operand right before its product)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[i % AHEAD].v, q[i / 2].v, s[i % 2], 0, 0, 0);
      if (i + AHEAD < 8) load_k(i + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // max3 below is a statement of its own, before which the compiler does not wait for a matrix product's result: 19
    // states after one of 16 passes.
    asm volatile("s_nop 15\n s_nop 7" : "+v"(s[0]), "+v"(s[1]));
    if constexpr (SCALED) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const f32x4 as = *reinterpret_cast<const f32x4*>(&scales[buf][0][32 * kb + 8 * (i / 4) + 4 * half + i % 4]);
          s[kb][i] = __builtin_fmaf(as[1], s[kb][i], as[0] * q_sum);
          s[kb][i + 1] = __builtin_fmaf(as[3], s[kb][i + 1], as[2] * q_sum);
        }
    }
    if (masked) {
      const int below = high - 4 * half;  // (compared with constants: the lanes' keys are not kept in registers)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i / 4) + i % 4 < below ? s[kb][i] : -INFINITY;
    }
    float top = max3(s[0][0], s[0][1], s[0][2]), top1 = max3(s[1][0], s[1][1], s[1][2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) top = max3(top, s[0][i], s[0][i + 1]), top1 = max3(top1, s[1][i], s[1][i + 1]);
    top = max_nn(max3(top, s[0][15], s[1][15]), top1);
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
    for (int kb = 0; kb < 2; ++kb) {
      if (kb == 1 && one_half) break;  // (8 frames of 78 tokens, 3 terms: 80 us with it, 86 without; full units 1 % either way)
#pragma unroll
      for (int st = 0; st < 2; ++st) {  // 16 keys
        Op8 p[TERMS], v[2];
        if (PREC) __builtin_amdgcn_sched_barrier(0);  // (8 frames 80 us with it, 82 without: the scales of all keys are read first)
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            v[db].h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(vt + (v_at ^ (64 * db) ^ (32 * j)) + (32 * kb + 16 * st + 8 * j) * 128));
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * st + j], xs, -mref));
          float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * st + j + 1], xs, -mref));
          if (TERMS > 1) sum += p0 + p1;
          if constexpr (SCALED) {
            const f32x4 as = *reinterpret_cast<const f32x4*>(&scales[buf][1][32 * kb + 16 * st + 8 * (j / 4) + 4 * half + j % 4]);
            offset = __builtin_fmaf(p0, as[0], offset);
            offset = __builtin_fmaf(p1, as[2], offset);
            p0 *= as[1], p1 *= as[3];
          }
          uint32_t x[TERMS];
          split_pair<TERMS>(p0, p1, x);
#pragma unroll
          for (int k = 0; k < TERMS; ++k) p[k].u[j / 2] = x[k];
          // (Weights of one bf16 value are summed as they are multiplied.)
          if (TERMS == 1) sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x[0]), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
        }
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
          for (int k = TERMS - 1; k >= 0; --k) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[db].v, p[k].v, acc[db], 0, 0, 0);
      }
    }
    l_part += sum;
  };
  // What was asked for before this iteration has landed (this wave's part; the barrier: every wave's), the next unit is
  // unpacked, and no wave reads this one any more.
  auto step = [&](int asked) {
    wait_loads(asked);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  int buf = 0, u = w.u0;
  for (; u < min(w.u1, w.n_pages); ++u) {
    const int next = buf + 1 == RING ? 0 : buf + 1, after = next + 1 == RING ? 0 : next + 1;
    int asked = 0;  // loads of this wave in this iteration
    if (x3.bits < 16) load_raw(x3, buf), asked = x3.loads;  // (unit u's packed rows were unpacked in the iteration before)
    if (x2.bits == 16 && x2.rows) load_tile(u + 2, x2, after), asked += x2.loads;
    if (x1.bits < 16) unpack(x1, next, next);
    const Unit x4 = unit_at(u + 4);
    if (x0.rows < TILE && x0.bits == 16) zero_values(x0, tiles[buf][1], false);
    if (on) attend(std::integral_constant<bool, PREC == 1>(), buf, x0.rows < TILE, x0.rows, x0.rows <= 32);
    step(asked);
    x0 = x1, x1 = x2, x2 = x3, x3 = x4;
    buf = next;
  }
  const int m_new = min(wave0 + (anew(t) & 31), total - 1) / G;  // this lane's token again
  const uint8_t* kn = new_rows(a.k_new, a.kn_head_stride, a.kn_tok_stride, u + 2);
  const uint8_t* vn = new_rows(a.v_new, a.vn_head_stride, a.vn_tok_stride, u + 2);
  for (; u < w.u1; ++u) {  // new tokens: nothing to be unpacked
    const int next = buf + 1 == RING ? 0 : buf + 1, after = next + 1 == RING ? 0 : next + 1;
    const int first = (u - w.n_pages) * TILE;
    const bool more = u + 2 < w.u1;
    if (more) load_rows(std::false_type(), kn, vn, w.count - first - 2 * TILE, kn_stride, vn_stride, after);
    kn += 2 * TILE * a.kn_tok_stride, vn += 2 * TILE * a.vn_tok_stride;
    if (first + TILE - 1 > first_token) zero_values(Unit{16, min(TILE, w.count - first), 0, 0}, tiles[buf][1], true);
    if (on && first <= m_last) attend(std::false_type(), buf, first + TILE - 1 > m_first, m_new + 1 - first, m_last - first < 32);
    step(more ? 2 : 0);
    buf = next;
  }
  if (!on) return;
  const int last = anew(t), c_last = last & 31, half_last = last >> 5 & 1, row_last = min(wave0 + c_last, total - 1), m_out = row_last / G;
  auto both = [](float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
  };
  const float l = both(l_part), off = PREC ? both(offset) : 0.f;
  // (rare) New values that the products took for zero, with their weights computed again; where an element of this wave became NaN,
  // which an infinite value's products with a weight's lower terms also make, all infinite and NaN values that it sees.
  uint32_t lost = 0;  // such elements, of rows whose scores are no NaN: bit 16 db + i
  if (TERMS > 1)
#pragma unroll
    for (int i = 0; i < 32; ++i) lost |= acc[i / 16][i % 16] != acc[i / 16][i % 16] && l == l ? 1u << i : 0u;
  const bool again = TERMS > 1 && __builtin_amdgcn_ballot_w64(lost != 0);
  if (bad || again) {
    asm volatile("" : "+v"(q[0].u), "+v"(q[1].u), "+v"(q[2].u), "+v"(q[3].u));  // (as values of their own, as in anew)
    if (TERMS > 1)
#pragma unroll
      for (int i = 0; i < 32; ++i) acc[i / 16][i % 16] = lost >> i & 1 ? 0.f : acc[i / 16][i % 16];
    bool packed = false;  // a packed row of values is infinite or NaN: its elements stay NaN
    for (int u = again ? w.u0 : max(w.u0, w.n_pages); u < w.u1; ++u) {
      const int first = (u - w.n_pages) * TILE;
      const uint8_t *k, *v;
      int64_t k_stride = 128, v_stride = 128;
      int rows;
      if (u < w.n_pages) {
        const Page pg = plan_record<Page>(plan, a.plan.at_pages, w.first_page + u);
        const int bits = page_bits(pg.page);
        k = base + (pg.page >> 2) * grain + sub * page_sub(bits), v = k + (int64_t)H * page_sub(bits), rows = pg.rows;
        if (bits < 16) {
          const float2 as = reinterpret_cast<const float2*>(v + TILE * 8 * bits)[last & 63];
          packed = packed || ((last & 63) < rows && !(fabsf(as.x) < INFINITY && fabsf(as.y) < INFINITY));
          continue;
        }
      } else {
        if (!again && first + TILE - 1 <= first_token) continue;
        k = new_rows(a.k_new, a.kn_head_stride, a.kn_tok_stride, u), v = new_rows(a.v_new, a.vn_head_stride, a.vn_tok_stride, u);
        k_stride = 2 * a.kn_tok_stride, v_stride = 2 * a.vn_tok_stride, rows = min(TILE, w.count - first);
      }
      for (int j = 0; j < rows; ++j, k += k_stride, v += v_stride) {
        uint2 x[8];
        bool some = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // elements 8 i + 4 half_last + ...
          x[i] = reinterpret_cast<const uint2*>(v)[2 * i + half_last];
          some = some || bad_bf16(x[i].x) || bad_bf16(x[i].x >> 16) || bad_bf16(x[i].y) || bad_bf16(x[i].y >> 16);
        }
        if (!__builtin_amdgcn_ballot_w64(some)) continue;
        float dot = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const u32x4 y = reinterpret_cast<const u32x4*>(k)[2 * ks + half_last];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dot = __builtin_fmaf(bf16_lo(q[ks].u[e]), bf16_lo(y[e]), __builtin_fmaf(bf16_hi(q[ks].u[e]), bf16_hi(y[e]), dot));
        }
        const float p = __builtin_amdgcn_exp2f(both(dot) * xs - m_run);
        if (first + j > m_out) continue;  // (of pages: negative)
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
    if (TERMS > 1) {
      const bool keep = __builtin_amdgcn_ballot_w64(packed);
#pragma unroll
      for (int i = 0; i < 32; ++i)  // (no such value was found: the NaN comes from a score)
        if (lost >> i & 1 && (keep || acc[i / 16][i % 16] == 0.f)) acc[i / 16][i % 16] = NAN;
    }
  }
  if (wave0 + c_last >= total) return;
  if (w.part < 0) {
    const float inv = 1.f / l;
    const int64_t at = (int64_t)(w.token0 + m_out) * a.out_tok_stride + (int64_t)(h * G + row_last - m_out * G) * a.out_head_stride + 4 * half_last;
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const f32x4 x = f32x4{acc[i / 16][i % 16] + off, acc[i / 16][i % 16 + 1] + off, acc[i / 16][i % 16 + 2] + off, acc[i / 16][i % 16 + 3] + off} * inv;
      store4(a.out, a.out_dtype, at + 32 * (i / 16) + 8 * (i % 16 / 4), x);
    }
  } else {
    const int64_t at = (int64_t)(w.part + 32 * wave + c_last) * H + h;
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<f32x4*>(part_o + at * D + 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * half_last) =
          f32x4{acc[i / 16][i % 16] + off, acc[i / 16][i % 16 + 1] + off, acc[i / 16][i % 16 + 2] + off, acc[i / 16][i % 16 + 3] + off};
    if (half_last == 0) part_ml[at] = make_float2(m_run, l);
  }
}

void launch_long(const dkv_paged_args& a, int n_long, int n_short, float* part_o, float2* part_ml, hipStream_t s) {
  const auto kernel = a.precision == 1 ? long_kernel<1, 3, 3> : a.out_dtype == 1 ? long_kernel<0, 3, 3> : long_kernel<0, 1, 2>;
  hipLaunchKernelGGL(kernel, dim3((n_long + n_short) * a.plan.heads), dim3(64 * WAVES), 0, s, a, n_long, part_o, part_ml);
}

}  // namespace paged
}  // namespace dkv
