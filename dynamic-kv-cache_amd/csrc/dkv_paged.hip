// Paged caches of many sequences (gfx950): a step's plan, the pack of its new rows, pages read back, rows moved.
//
// A plan is made on the host once a step and read by every layer's launches, so no kernel searches a table: a workgroup
// loads one record that names its pages, rows and share of the work.
#include "dkv_paged.h"
#include "dkv_rope_pack.h"
#include <string.h>
#include <algorithm>
#include <functional>
#include <new>
#include <vector>

namespace dkv {
namespace paged {

// ---- the pack ----------------------------------------------------------------------------------------------------

// A row held by 8 lanes (lane c: elements [8 c, 8 c + 8)) into a page, with dkv_pack's arithmetic.
template <int BITS>
__device__ __forceinline__ void pack_row(const u32x4& w, bool valid, int c, uint8_t* sub, int row) {
  if (BITS == 16) {
    if (valid) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(sub + row * 128 + 16 * c));
    return;
  }
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[2 * e] = bf16_lo(w[e]), x[2 * e + 1] = bf16_hi(w[e]);
  float lo = x[0], hi = x[0];
  uint32_t nz = 0;  // the row holds a -0 (zero_min_sign)
#pragma unroll
  for (int e = 0; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]), nz |= __float_as_uint(x[e]) == 0x80000000u;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, o));
    hi = fmaxf(hi, __shfl_xor(hi, o));
    nz |= __shfl_xor(nz, o);
  }
  const float a = lo == 0.0f ? zero_min_sign(nz) : lo;
  const float span = hi - a;
  const float s = span > 0.0f ? __fdiv_rn(span, BITS == 4 ? 15.0f : 255.0f) : 1.0f;
  const float rs = __builtin_amdgcn_rcpf(s);
  const bool fast = s >= 0x1p-126f && s <= 0x1p125f;
  uint32_t out[2];
  quantize8<BITS>(x, a, s, rs, fast, out);
  if (!valid) return;
  if (BITS == 4) __builtin_nontemporal_store(out[0], reinterpret_cast<uint32_t*>(sub + row * 32 + 4 * c));
  else __builtin_nontemporal_store((uint64_t)out[1] << 32 | out[0], reinterpret_cast<uint64_t*>(sub + row * 64 + 8 * c));
  if (c == 0)
    __builtin_nontemporal_store((uint64_t)__float_as_uint(s) << 32 | __float_as_uint(a),
                                reinterpret_cast<uint64_t*>(sub + TILE * 8 * BITS + 8 * row));
}

// Rows r0 + 8 i of at most HALF_ITEM, 8 lanes a row, all loaded before the first is packed.
constexpr int HALF_ITEM = 32;
template <int BITS>
__device__ __forceinline__ void pack_rows(const uint16_t* src, int64_t stride, int rows, int r0, int c, uint8_t* sub, int row0) {
  u32x4 w[HALF_ITEM / 8];
#pragma unroll
  for (int i = 0; i < HALF_ITEM / 8; ++i) w[i] = *reinterpret_cast<const u32x4*>(src + min(8 * i + r0, rows - 1) * stride + 8 * c);
#pragma unroll
  for (int i = 0; i < HALF_ITEM / 8; ++i) {
    if (8 * i >= rows) break;
    pack_row<BITS>(w[i], 8 * i + r0 < rows, c, sub, row0 + 8 * i + r0);
  }
}

// Packs a step's rows: a = min, s = (max - min) / (2^b - 1), q = rint((x - a) / s), dkv_pack's bytes. Bound by the bytes of a long
// prompt (128 read and 40 to 136 written a row) and the launch of a short one. A wave takes half of the rows of one item (up to 64
// tokens of a page) of one K or V head, whose loads are one group: 5833 tokens of 8 heads, 21.9 MB, 8.2 us (2.7 TB/s; whole items in
// two groups 10.5, in one, which takes 230 registers, 13.6), a token of each of 32 sequences of 5 heads 2.8 us.
__global__ __launch_bounds__(256) void append_kernel(dkv_paged_args a) {
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  if (a.bounds && (int)(blockIdx.x >> 1) >= plan[N_ITEMS]) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, H = a.plan.heads;
  const int kvh = blockIdx.y * 4 + wave;
  if (kvh >= 2 * H) return;
  dkv_page_rows item = plan_record<dkv_page_rows>(plan, a.plan.at_items, blockIdx.x >> 1);
  const int skip = HALF_ITEM * (blockIdx.x & 1);
  if (skip >= item.rows) return;
  item.token += skip, item.row0 += skip, item.rows = min(HALF_ITEM, item.rows - skip);
  const int kv = kvh >= H, h = kvh - kv * H, c = lane & 7, r0 = lane >> 3;
  const uint16_t* src = static_cast<const uint16_t*>(kv ? a.v_new : a.k_new) +
                        (kv ? h * a.vn_head_stride + item.token * a.vn_tok_stride : h * a.kn_head_stride + item.token * a.kn_tok_stride);
  const int64_t stride = kv ? a.vn_tok_stride : a.kn_tok_stride;
  const int bits = page_bits(item.page);
  uint8_t* sub = static_cast<uint8_t*>(a.arena) + page_at(item.page, a.layer, a.plan.layers, H, 0) + (int64_t)kvh * page_sub(bits);
  if (bits == 4) pack_rows<4>(src, stride, item.rows, r0, c, sub, item.row0);
  else if (bits == 8) pack_rows<8>(src, stride, item.rows, r0, c, sub, item.row0);
  else pack_rows<16>(src, stride, item.rows, r0, c, sub, item.row0);
}

// The joined projection's rows [q | k | v] of one item and head: rotated (Q and K heads; V rows keep their input), stored,
// and for K and V heads packed. 8 lanes a row as above; rotate_half pairs lane c with lane c ^ 4. (A token of each of 4 / 48
// sequences, 15 + 2 * 5 heads: one launch of 3.6 / 3.8 us in place of RoPE's 2.8 / 3.2 and the pack's 2.5 / 3.2; 24 prompts of 6503 tokens
// together 18.4 us, 48 MB at 2.6 TB/s, in place of 21.2 for both.)
template <int BITS>
__device__ __forceinline__ void rope_rows(const uint16_t* src, int64_t src_stride, const uint16_t* cosv, const uint16_t* sinv, int64_t cs_stride,
                                          int rows, int r0, int c, bool is_v, uint16_t* dst, int64_t dst_stride, uint8_t* sub, int row0) {
  constexpr int AHEAD = 2;
  for (int i0 = 0; i0 < rows; i0 += 8 * AHEAD) {
    u32x4 x[AHEAD], cs[AHEAD], sn[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int row = min(i0 + 8 * i + r0, rows - 1);
      x[i] = *reinterpret_cast<const u32x4*>(src + row * src_stride + 8 * c);
      cs[i] = *reinterpret_cast<const u32x4*>(cosv + row * cs_stride + 8 * c);
      sn[i] = *reinterpret_cast<const u32x4*>(sinv + row * cs_stride + 8 * c);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int row = i0 + 8 * i + r0;
      if (i0 + 8 * i >= rows) break;
      u32x4 p;
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = __shfl_xor(x[i][e], 4);
      const u32x4 rot = rope8(x[i], p, cs[i], sn[i], c < 4), w = is_v ? x[i] : rot;
      if (row < rows) *reinterpret_cast<u32x4*>(dst + row * dst_stride + 8 * c) = w;
      if (BITS) pack_row<BITS ? BITS : 16>(w, row < rows, c, sub, row0 + row);
    }
  }
}

__global__ __launch_bounds__(256) void rope_append_kernel(dkv_paged_args a, const uint16_t* qkv, int64_t qkv_stride, const uint16_t* cosv,
                                                          const uint16_t* sinv, int64_t cs_stride) {
  const int32_t* plan = static_cast<const int32_t*>(a.plan_words);
  if (a.bounds && (int)blockIdx.x >= plan[N_ITEMS]) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, H = a.plan.heads, Hq = a.plan.q_heads;
  const int hh = blockIdx.y * 4 + wave;  // of Q, then K, then V
  if (hh >= Hq + 2 * H) return;
  const dkv_page_rows item = plan_record<dkv_page_rows>(plan, a.plan.at_items, blockIdx.x);
  const int kvh = hh - Hq, kv = kvh >= H, h = kvh - kv * H, c = lane & 7, r0 = lane >> 3;
  const uint16_t* src = qkv + item.token * qkv_stride + hh * D;
  const uint16_t *cs = cosv + item.token * cs_stride, *sn = sinv + item.token * cs_stride;
  if (kvh < 0) {
    uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(a.q)) + hh * a.q_head_stride + item.token * a.q_tok_stride;
    rope_rows<0>(src, qkv_stride, cs, sn, cs_stride, item.rows, r0, c, false, dst, a.q_tok_stride, nullptr, 0);
    return;
  }
  const int64_t stride = kv ? a.vn_tok_stride : a.kn_tok_stride;
  uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(kv ? a.v_new : a.k_new)) + h * (kv ? a.vn_head_stride : a.kn_head_stride) + item.token * stride;
  const int bits = page_bits(item.page);
  uint8_t* sub = static_cast<uint8_t*>(a.arena) + page_at(item.page, a.layer, a.plan.layers, H, 0) + (int64_t)kvh * page_sub(bits);
  if (bits == 4) rope_rows<4>(src, qkv_stride, cs, sn, cs_stride, item.rows, r0, c, kv, dst, stride, sub, item.row0);
  else if (bits == 8) rope_rows<8>(src, qkv_stride, cs, sn, cs_stride, item.rows, r0, c, kv, dst, stride, sub, item.row0);
  else rope_rows<16>(src, qkv_stride, cs, sn, cs_stride, item.rows, r0, c, kv, dst, stride, sub, item.row0);
}

// ---- pages read back ---------------------------------------------------------------------------------------------

constexpr int ARG_ITEMS = 224;  // records of a launch's argument block, of less than 4 KB
struct Items {
  dkv_page_rows at[ARG_ITEMS];
};

// Rows of a page as values code * s + a, 8 lanes a row (lane c: elements [8 c, 8 c + 8)): every store of bf16 writes whole lines.
// Bound by its bytes: 8138 tokens of 8 layers of 5 heads, 131 MB read and written, 25.5 us (5.1 TB/s; in launches of 128 records
// 31).
template <int BITS>
__device__ __forceinline__ void read_rows(const uint8_t* sub, int row0, int rows, int r0, int c, void* out, int64_t at, int out_dtype) {
  constexpr int AHEAD = 4;
  for (int i0 = 0; i0 < rows; i0 += 8 * AHEAD) {
    u32x4 w[AHEAD];
    float2 as[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int row = row0 + min(i0 + 8 * i + r0, rows - 1);
      const uint8_t* p = sub + row * (8 * BITS) + c * BITS;
      if (BITS == 4) w[i][0] = *reinterpret_cast<const uint32_t*>(p);
      else if (BITS == 16) w[i] = *reinterpret_cast<const u32x4*>(p);
      else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[i][0] = x.x, w[i][1] = x.y;
      }
      if (BITS < 16) as[i] = reinterpret_cast<const float2*>(sub + TILE * 8 * BITS)[row];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int r = i0 + 8 * i + r0;
      if (r >= rows) break;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (BITS == 16) x[e] = e & 1 ? bf16_hi(w[i][e / 2]) : bf16_lo(w[i][e / 2]);
        else x[e] = __fadd_rn(__fmul_rn((float)(BITS == 4 ? (w[i][0] >> (4 * e)) & 15u : (w[i][e / 4] >> (8 * (e % 4))) & 255u), as[i].y), as[i].x);
      }
      const int64_t o = at + (int64_t)r * D + 8 * c;
      if (out_dtype == 1) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + o);
        dst[0] = make_float4(x[0], x[1], x[2], x[3]), dst[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + o) =
            u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
      }
    }
  }
}

// A wave: the rows of one item of one (layer, K or V, head).
__global__ __launch_bounds__(256) void read_kernel(Items items, const uint8_t* __restrict__ arena, int layer0, int n_layers, int layers,
                                                   int heads, void* __restrict__ out, int64_t n_tokens, int out_dtype) {
  const dkv_page_rows item = items.at[blockIdx.x];
  const int sub_index = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  if (sub_index >= 2 * heads * n_layers) return;
  const int l = sub_index / (2 * heads), kvh = sub_index - l * 2 * heads, kv = kvh >= heads, h = kvh - kv * heads;
  const int bits = page_bits(item.page);
  const uint8_t* sub = arena + page_at(item.page, layer0 + l, layers, heads, 0) + (int64_t)kvh * page_sub(bits);
  const int64_t at = ((((int64_t)kv * n_layers + l) * heads + h) * n_tokens + item.token) * D;
  if (bits == 4) read_rows<4>(sub, item.row0, item.rows, lane >> 3, lane & 7, out, at, out_dtype);
  else if (bits == 8) read_rows<8>(sub, item.row0, item.rows, lane >> 3, lane & 7, out, at, out_dtype);
  else read_rows<16>(sub, item.row0, item.rows, lane >> 3, lane & 7, out, at, out_dtype);
}

// ---- rows moved --------------------------------------------------------------------------------------------------

constexpr int ARG_MOVES = 160;
struct Moves {
  dkv_page_move at[ARG_MOVES];
};

// One sub-block's rows: the payload in 16-byte pieces, then the (offset, scale) pairs, which lie behind as many rows as
// the tile has room for. All loads before the first store. Bound by its bytes: the same history gathered into pages, 96 MB, some 25 us
// in two launches, of 160 and 100 moves (3.9 TB/s).
template <int BITS>
__device__ __forceinline__ void move_rows(const dkv_page_move& m, const uint8_t* from, uint8_t* to, int lane) {
  constexpr int ROW = 8 * BITS, PIECES = BITS / 2;  // bytes; of 64 rows, a lane's pieces
  const u32x4* f = reinterpret_cast<const u32x4*>(from + m.src_row * ROW);
  u32x4* t = reinterpret_cast<u32x4*>(to + m.dst_row * ROW);
  const int n = m.rows * (ROW / 16);
  u32x4 w[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) w[i] = f[min(64 * i + lane, n - 1)];
  uint2 as = make_uint2(0, 0);
  if (BITS < 16) as = reinterpret_cast<const uint2*>(from + m.src_rows * ROW)[m.src_row + min(lane, m.rows - 1)];
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
    if (64 * i + lane < n) __builtin_nontemporal_store(w[i], t + 64 * i + lane);
  if (BITS < 16 && lane < m.rows) reinterpret_cast<uint2*>(to + TILE * ROW)[m.dst_row + lane] = as;
}

// A wave moves the rows of one (layer, K or V, head) of a move.
__global__ __launch_bounds__(256) void move_kernel(Moves moves, const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, int subs) {
  const dkv_page_move m = moves.at[blockIdx.x];
  const int sub = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  if (sub >= subs) return;
  const uint8_t* from = src + m.src_offset + sub * subblock_bytes(m.src_rows, m.bits);
  uint8_t* to = dst + m.dst_offset + (int64_t)sub * page_sub(m.bits);
  if (m.bits == 4) move_rows<4>(m, from, to, lane);
  else if (m.bits == 8) move_rows<8>(m, from, to, lane);
  else move_rows<16>(m, from, to, lane);
}

int launch_moves(const void* src, void* dst, const dkv_page_move* moves, int n_moves, int layers, int heads, void* stream) {
  if (!dst) return 0;
  const int subs = 2 * layers * heads;
  for (int i = 0; i < n_moves; i += ARG_MOVES) {
    const int n = std::min(ARG_MOVES, n_moves - i);
    Moves block{};
    memcpy(block.at, moves + i, n * sizeof(dkv_page_move));
    hipLaunchKernelGGL(move_kernel, dim3(n, (subs + 3) / 4), dim3(256), 0, (hipStream_t)stream, block, static_cast<const uint8_t*>(src),
                       static_cast<uint8_t*>(dst), subs);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  return 0;
}

// ---- plans -------------------------------------------------------------------------------------------------------

// Entities of up to this many query rows of a KV head go to the kernel for few rows. In us there / in the kernel for many, single tokens
// of branches: 5 heads of 3 over 127 pages in common, bf16, 96 rows 15.5 / 16.8, 144 19.1 / 19.4, 162 21.3 / 20.0, 258 28.0 / 25.3; 8 heads of
// 4 over 32 pages 96 rows 12.6 / 12.7, 164 16.3 / 14.8, 320 22.0 / 22.2; over 625 pages 96 rows 41.2 / 33.6, 162 61.7 / 39.7. At precision 1,
// whose kernel for many splits weights in three, few rows stay ahead for longer: 162 rows over the 127 pages 20.5 / 28.1, 321 30.6 / 35.1.
// 16 questions of 15 to 180 rows about 96 pages, few rows in a launch of their own: 40.6 us by this rule, 43.5 from 100 rows on, 40.9 from 200.
constexpr int SHORT_ROWS = 160;
// Few rows (four waves, a unit each at a time): about SHORT_TARGET workgroups over all KV heads share a step's units, four
// resident a CU, of SHORT_LEAST units at least (three short histories 8.4 us with 8, 12.1 with 4 and a join). A token of 64
// streams / of 6 long ones: 1024 workgroups 34.3 / 113 us, 2048 31.7 / 106.
constexpr int SHORT_TARGET = 2048, SHORT_LEAST = 8;
// Many rows (eight waves, a unit at a time): a step is split into LONG_TARGET workgroups at most (two a CU) beside those that
// its blocks need, of LONG_LEAST units at least, by ranges of such a length that the last workgroup ends first (long_share).
constexpr int LONG_TARGET = 512, LONG_LEAST = 2, SLOTS[2] = {256, 512};
constexpr int SHARED_MIN = 4;  // pages that neighbours have in common to be attended to as a group

struct Entity {  // a sequence's own part, or what a group of sequences has in common
  int first_page, n_pages, token0, count;
  int n4, n8;  // pages up to which they have 4 bits, 8 at most
  bool group;
  int64_t part;  // of a group: its first partial row
  int splits;
};

static int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

static bool is_long(int64_t rows) { return rows > SHORT_ROWS; }

static int check_batch(const dkv_paged_batch& b, const char* what) {
  if (b.seqs <= 0 || !b.count || !b.past || !b.position || !b.first || b.layers <= 0 || b.heads <= 0 || b.q_heads <= 0 ||
      b.q_heads % b.heads || b.max_pages < 0 || b.precision < 0 || b.precision > 1) {
    set_error("%s: bad batch (seqs %d, layers %d, heads %d, q_heads %d) or a null array", what, b.seqs, b.layers, b.heads, b.q_heads);
    return DKV_EINVAL;
  }
  if ((int64_t)b.layers * b.heads > 65535 / 2 || b.heads > 16384 || b.q_heads / b.heads > 4096) {
    set_error("%s: too many layers or heads (%d layers, %d of %d heads)", what, b.layers, b.heads, b.q_heads);
    return DKV_EINVAL;
  }
  int64_t tokens = 0;
  for (int i = 0; i < b.seqs; ++i) {
    if (b.count[i] <= 0 || b.past[i] < 0 || (int64_t)b.past[i] + b.count[i] > INT32_MAX) {
      set_error("%s: sequence %d has %d new tokens after %d", what, i, b.count[i], b.past[i]);
      return DKV_EINVAL;
    }
    tokens += b.count[i];
  }
  if (tokens * (b.q_heads / b.heads) > 1 << 24 || tokens > 1 << 22) {
    set_error("%s: %lld new tokens are too many for one step", what, (long long)tokens);
    return DKV_EINVAL;
  }
  return 0;
}

// The places and bounds of a plan of these counts, whatever the history.
static void layout_of(const dkv_paged_batch& b, dkv_paged_plan& p) {
  const int G = b.q_heads / b.heads;
  int64_t tokens = 0, items = 0, merges = 0, few = 0, many = 0;  // blocks of few and of many rows
  for (int i = 0; i < b.seqs; ++i) {
    const int64_t rows = (int64_t)b.count[i] * G;
    tokens += b.count[i];
    items += ceil_div(b.count[i], TILE) + 1;
    merges += ceil_div(rows, SHORT_BLOCK);
    if (is_long(rows)) many += ceil_div(rows, LONG_BLOCK);
    else few += ceil_div(rows, SHORT_BLOCK);
  }
  if (b.seqs > 1) {  // groups: of all tokens together, each of two sequences at least
    const int64_t rows = tokens * G;
    few += ceil_div(std::min<int64_t>(rows, (int64_t)b.seqs / 2 * SHORT_ROWS), SHORT_BLOCK) + b.seqs / 2;
    if (is_long(rows)) many += ceil_div(rows, LONG_BLOCK) + std::min<int64_t>(b.seqs / 2, rows / SHORT_ROWS);
  }
  p.seqs = b.seqs, p.tokens = (int)tokens, p.layers = b.layers, p.heads = b.heads, p.q_heads = b.q_heads;
  p.grains = (int)std::min<int64_t>(std::max<int64_t>(b.arena_bytes, 0) / grain_bytes(b.layers, b.heads), 1 << 30);
  p.max_items = (int)items;
  p.max_pages = b.max_pages;
  p.max_work = few ? (int)(few + ceil_div(SHORT_TARGET, b.heads)) : 0;
  p.max_long = many ? (int)(many + ceil_div(LONG_TARGET, b.heads)) : 0;
  p.max_merges = (int)merges;
  p.max_rows = p.max_work * SHORT_BLOCK + p.max_long * LONG_BLOCK;
  auto up = [](int64_t x) { return (x + 15) & ~(int64_t)15; };
  int64_t at = HEAD_WORDS;
  p.at_items = (int)at, at += up(4 * items);
  p.at_positions = (int)at, at += up(2 * tokens);
  p.at_pages = (int)at, at += up(2 * (int64_t)b.max_pages);
  p.at_work = (int)at, at += up((int64_t)(sizeof(Work) / 4) * p.max_work);
  p.at_long = (int)at, at += up((int64_t)(sizeof(Work) / 4) * p.max_long);
  p.at_merges = (int)at, at += up(8ll * p.max_merges);
  p.words = (int)at;
}

// A batch whose plan's offsets fit into 32 bits, and its launches' threads.
static int check_plan(const dkv_paged_batch& b, const char* what) {
  if (int rc = check_batch(b, what)) return rc;
  int64_t tokens = 0;
  for (int i = 0; i < b.seqs; ++i) tokens += b.count[i];
  bool fits = 64 * tokens * (b.q_heads / b.heads) + 64ll * b.seqs + 2ll * b.max_pages + (1 << 20) < INT32_MAX;
  if (fits) {
    dkv_paged_plan p{};
    layout_of(b, p);
    const int64_t threads = std::max<int64_t>({2ll * p.max_items, (int64_t)p.max_work * b.heads, 2ll * (p.max_long + p.max_work) * b.heads,
                                      (int64_t)p.max_merges * (SHORT_BLOCK / 4) * b.heads}) * 256;
    fits = threads <= UINT32_MAX;
  }
  if (fits) return 0;
  set_error("%s: %lld new tokens, %d query heads and %d pages are too many for one step", what, (long long)tokens, b.q_heads, b.max_pages);
  return DKV_EINVAL;
}

// Units that a block of an entity's query rows sees: a group's pages, or a sequence's and its new tokens up to the
// block's last one.
static int units_of(const Entity& e, int G, int block, int blk) {
  if (e.group) return e.n_pages;
  const int last = (int)std::min<int64_t>(((int64_t)(blk + 1) * block - 1) / G, e.count - 1);
  return e.n_pages + last / TILE + 1;
}

static int64_t total_units(const std::vector<Entity>& es, int G, bool many) {
  const int block = many ? LONG_BLOCK : SHORT_BLOCK;
  int64_t total = 0;
  for (const Entity& e : es)
    if (is_long((int64_t)e.count * G) == many)
      for (int blk = 0, n = ceil_div((int64_t)e.count * G, block); blk < n; ++blk) total += units_of(e, G, block, blk);
  return total;
}

// Units of a workgroup so that about `target` of them a KV head share all entities' units of this kind.
static int64_t share(int64_t total, int64_t target, int least) { return std::max<int64_t>(least, (total + target - 1) / target); }

// The same for many rows: of ranges from that length on, the one whose workgroups are done first when each free place takes the
// longest that is left. A CU is one place, since one workgroup keeps its vector units busy; at precision 1 it is two (8 frames 83 us,
// 104 with one). In units: a workgroup costs its units and what its start takes, one that is joined its partial rows beside, and the
// join reads them. (Equal shares for 512 workgroups and for 256: 12500 tokens of prompts 228 and 204 us, 12 prompts 73.8 and 59.4, 16
// questions 42.6 and 40.6; these 204, 59.4 and 40.7, all with few rows in a launch of their own.)
static int64_t long_share(const std::vector<Entity>& es, int G, int heads, int precision, int groups, const std::vector<int>& group) {
  const int slots = std::max(1, SLOTS[precision] / heads);
  const int64_t least = share(total_units(es, G, true), ceil_div(LONG_TARGET, heads), LONG_LEAST);
  int64_t most = 0, best = least;
  for (const Entity& e : es)
    if (is_long((int64_t)e.count * G)) most = std::max<int64_t>(most, units_of(e, G, LONG_BLOCK, ceil_div((int64_t)e.count * G, LONG_BLOCK) - 1));
  constexpr float START = 1.f, PARTIAL = 2.f, JOIN = 3e-5f;  // of a workgroup; of its 256 rows; of a partial row and head
  float best_time = 0.f;
  std::vector<float> costs, ends;
  for (int64_t len = least;; len += std::max<int64_t>(1, len / 4)) {
    costs.clear();
    int64_t rows = 0;
    for (size_t i = 0; i < es.size(); ++i) {
      const Entity& e = es[i];
      const int64_t total = (int64_t)e.count * G;
      if (!is_long(total)) continue;
      for (int blk = 0; blk < ceil_div(total, LONG_BLOCK); ++blk) {
        const int units = units_of(e, G, LONG_BLOCK, blk), splits = std::max(1, ceil_div(units, len));
        const bool parts = splits > 1 || e.group || group[i - groups] >= 0;
        if (parts) rows += (int64_t)splits * std::min<int64_t>(LONG_BLOCK, total - (int64_t)blk * LONG_BLOCK);
        for (int s = 0; s < splits; ++s) costs.push_back((float)units / splits + START + (parts ? PARTIAL : 0.f));
      }
    }
    std::sort(costs.begin(), costs.end(), std::greater<float>());
    ends.assign(slots, 0.f);  // a heap of when each place is free
    float last = 0.f;
    for (float c : costs) {
      std::pop_heap(ends.begin(), ends.end(), std::greater<float>());
      last = std::max(last, ends.back() += c);
      std::push_heap(ends.begin(), ends.end(), std::greater<float>());
    }
    const float time = last + JOIN * (float)rows * heads;
    if (best_time == 0.f || time < best_time) best_time = time, best = len;
    if (len >= most) return best;
  }
}

static int write_plan(const dkv_paged_batch& b, int32_t* w, dkv_paged_plan& p) {
  const int G = b.q_heads / b.heads;
  layout_of(b, p);
  dkv_page_rows* items = reinterpret_cast<dkv_page_rows*>(w + p.at_items);
  Page* pages = reinterpret_cast<Page*>(w + p.at_pages);
  std::vector<Entity> own(b.seqs);
  int n_items = 0, n_pages = 0, token0 = 0;
  for (int i = 0; i < b.seqs; ++i) {
    const int from = b.first[i], to = b.first[i + 1];
    if (from < 0 || to < from || (to > from && (!b.page || !b.rows))) {
      set_error("dkv_paged_plan_write: sequence %d has pages [%d, %d)", i, from, to);
      return DKV_EINVAL;
    }
    Entity& e = own[i];
    e = Entity{n_pages, 0, token0, b.count[i], 0, 0, false, 0, 1};
    int64_t held = 0;
    const int64_t end = (int64_t)b.past[i] + b.count[i];
    for (int j = from; j < to; ++j) {
      const int code = b.page[j] & 3, rows = b.rows[j];
      if (code > 2 || (int64_t)(b.page[j] >> 2) + page_grains(4 << code) > p.grains) {
        set_error("dkv_paged_plan_write: page %u of sequence %d lies outside the arena", b.page[j], i);
        return DKV_EINVAL;
      }
      if (rows <= 0 || rows > TILE || held + rows > end) {
        set_error("dkv_paged_plan_write: a page of sequence %d has %d tokens after %lld of %lld", i, rows, (long long)held, (long long)end);
        return DKV_EINVAL;
      }
      const int old = (int)std::min<int64_t>(std::max<int64_t>(b.past[i] - held, 0), rows);
      if (old > 0) {
        if (n_pages >= b.max_pages) {
          set_error("dkv_paged_plan_write: the histories have more than the %d pages that the plan has room for", b.max_pages);
          return DKV_EINVAL;
        }
        pages[n_pages++] = Page{b.page[j], old};
        ++e.n_pages;
      }
      if (old < rows) {
        if (n_items >= p.max_items) {
          set_error("dkv_paged_plan_write: the %d new tokens of sequence %d lie in more pages than they need", b.count[i], i);
          return DKV_EINVAL;
        }
        items[n_items++] = dkv_page_rows{token0 + (int)(held + old - b.past[i]), b.page[j], old, rows - old};
      }
      held += rows;
    }
    if (held != end) {
      set_error("dkv_paged_plan_write: the pages of sequence %d hold %lld tokens, not %lld", i, (long long)held, (long long)end);
      return DKV_EINVAL;
    }
    int64_t* positions = reinterpret_cast<int64_t*>(w + p.at_positions) + token0;
    for (int t = 0; t < b.count[i]; ++t) positions[t] = (int64_t)b.position[i] + t;
    token0 += b.count[i];
  }
  // Neighbours that begin with the same pages attend to these as one entity, whose query rows are all their tokens'.
  std::vector<Entity> all;
  std::vector<int> group(b.seqs, -1);
  for (int i = 0; i < b.seqs;) {
    int same = 0, j = i + 1;
    for (; j < b.seqs; ++j) {
      const int most = std::min(j == i + 1 ? own[i].n_pages : same, own[j].n_pages);
      int n = 0;
      while (n < most && pages[own[i].first_page + n].page == pages[own[j].first_page + n].page &&
             pages[own[i].first_page + n].rows == pages[own[j].first_page + n].rows)
        ++n;
      if (n < SHARED_MIN || 2 * n < same) break;
      same = n;
    }
    if (same) {
      Entity g{own[i].first_page, same, own[i].token0, 0, 0, 0, true, 0, 1};
      for (int k = i; k < j; ++k) {
        g.count += own[k].count, group[k] = (int)all.size();
        own[k].first_page += same, own[k].n_pages -= same;
      }
      all.push_back(g);
    }
    i = j;
  }
  const int groups = (int)all.size();
  all.insert(all.end(), own.begin(), own.end());
  for (Entity& e : all) {  // by width (of pages that several sequences have in common, the first one's are read)
    Page* const from = pages + e.first_page;
    std::stable_sort(from, from + e.n_pages, [](const Page& x, const Page& y) { return (x.page & 3) < (y.page & 3); });
    for (int i = 0; i < e.n_pages; ++i) e.n4 += (from[i].page & 3) == 0, e.n8 += (from[i].page & 3) <= 1;
  }
  const int64_t few = share(total_units(all, G, false), ceil_div(SHORT_TARGET, b.heads), SHORT_LEAST);
  const int64_t many = long_share(all, G, b.heads, b.precision, groups, group);
  Work* const work = reinterpret_cast<Work*>(w + p.at_work);
  Work* const long_work = reinterpret_cast<Work*>(w + p.at_long);
  Merge* merges = reinterpret_cast<Merge*>(w + p.at_merges);
  int n_work = 0, n_long = 0, n_merges = 0;
  int64_t rows = 0, few_units = 0;  // partial rows so far; units of few query rows
  for (int i = 0; i < (int)all.size(); ++i) {
    Entity& e = all[i];
    const int64_t total = (int64_t)e.count * G;
    const bool is_many = is_long(total), joined = e.group || group[i - groups] >= 0;
    const int block = is_many ? LONG_BLOCK : SHORT_BLOCK, blocks = ceil_div(total, block);
    if (e.group) e.part = rows, e.splits = std::max(1, ceil_div(e.n_pages, is_many ? many : few)), rows += e.splits * total;
    for (int blk = 0; blk < blocks; ++blk) {
      const int units = units_of(e, G, block, blk), here = (int)std::min<int64_t>(block, total - (int64_t)blk * block);
      const int splits = e.group ? e.splits : std::max(1, ceil_div(units, is_many ? many : few));
      // a group's partial rows lie split after split, as its sequences' rows are not cut where its blocks are
      const int64_t first = e.group ? e.part + (int64_t)blk * block : rows, stride = e.group ? total : here;
      const bool parts = joined || splits > 1;
      if (!is_many) few_units += units;
      for (int s = 0; s < splits; ++s)
        (is_many ? long_work[n_long++] : work[n_work++]) =
            Work{e.first_page, e.n4, e.n8, e.n_pages, e.token0, e.count, blk, (int)((int64_t)units * s / splits),
                 (int)((int64_t)units * (s + 1) / splits), parts ? (int)(first + s * stride) : -1, {}};
      if (e.group || !parts) continue;
      rows += (int64_t)splits * here;
      for (int r = 0; r < here; r += SHORT_BLOCK) {
        Merge m{e.token0, (int)total, blk * block + r, (int)first + r, here, 0, 0, (uint32_t)splits};
        if (group[i - groups] >= 0) {
          const Entity& g = all[group[i - groups]];
          m.shared = (int)g.part + (e.token0 - g.token0) * G + m.row0, m.shared_stride = g.count * G, m.splits |= (uint32_t)g.splits << 16;
        }
        merges[n_merges++] = m;
      }
    }
  }
  auto longer = [](const Work& x, const Work& y) { return x.u1 - x.u0 > y.u1 - y.u0; };
  std::stable_sort(long_work, long_work + n_long, longer);  // (the longest first, so that none of them is left for the end)
  p.items = n_items, p.work = n_work, p.long_work = n_long, p.merges = n_merges, p.rows = (int)rows;
  p.units = (int)std::min<int64_t>(few_units, INT32_MAX);
  w[N_ITEMS] = n_items, w[N_WORK] = n_work, w[N_LONG] = n_long, w[N_MERGES] = n_merges;
  return 0;
}

int check_args(const dkv_paged_args& a, bool attend, const char* what) {
  const dkv_paged_plan& p = a.plan;
  auto a16 = [](const void* x) { return ((uintptr_t)x & 15) == 0; };
  if (!a.k_new || !a.v_new || !a.arena || !a.plan_words || (attend && (!a.q || !a.out))) {
    set_error("%s: null pointer argument", what);
  } else if (p.seqs <= 0 || p.tokens <= 0 || p.heads <= 0 || p.q_heads <= 0 || p.q_heads % p.heads || a.layer < 0 || a.layer >= p.layers) {
    set_error("%s: not a plan (seqs %d, heads %d of %d), or layer %d of %d", what, p.seqs, p.heads, p.q_heads, a.layer, p.layers);
  } else if (p.layers <= 0 || a.arena_bytes / grain_bytes(p.layers, p.heads) < p.grains) {
    set_error("%s: an arena of %lld bytes is smaller than the plan's of %d grains", what, (long long)a.arena_bytes, p.grains);
  } else if (!a16(a.k_new) || !a16(a.v_new) || !a16(a.arena) || !a16(a.plan_words) || (a.kn_head_stride & 7) || (a.kn_tok_stride & 7) ||
             (a.vn_head_stride & 7) || (a.vn_tok_stride & 7)) {
    set_error("%s: K, V, arena and plan must be 16-byte aligned with strides that are multiples of 8 elements", what);
  } else if (attend && (!a16(a.q) || !a16(a.out) || (a.q_head_stride & 7) || (a.q_tok_stride & 7) || (a.out_tok_stride & 3) ||
                        (a.out_head_stride & 3) || a.out_dtype < 0 || a.out_dtype > 1)) {
    set_error("%s: Q and out must be 16-byte aligned, strides multiples of 8 and 4 elements, out bf16 (0) or fp32 (1)", what);
  } else if (attend && (a.precision < 0 || a.precision > 1 || !(a.scale > 0.f) || a.scale > 3e38f)) {
    set_error("%s: precision must be 0 (bf16) or 1 (fp32), scale positive", what);
  } else if (attend && p.tokens > 1 && (a.kn_tok_stride < 0 || a.kn_tok_stride >= 1 << 23 || a.vn_tok_stride < 0 || a.vn_tok_stride >= 1 << 23)) {
    set_error("%s: K's and V's token strides must be from 0 to 2^23 - 1 elements", what);
  } else {
    return 0;
  }
  return DKV_EINVAL;
}

}  // namespace paged
}  // namespace dkv

using namespace dkv;
using namespace dkv::paged;

extern "C" {

int64_t dkv_page_grain(int32_t layers, int32_t heads) { return layers > 0 && heads > 0 ? grain_bytes(layers, heads) : 0; }

int64_t dkv_paged_plan_bytes(const dkv_paged_batch* batch) {
  clear_error();
  if (!batch) set_error("dkv_paged_plan_bytes: null batch");
  if (!batch || check_plan(*batch, "dkv_paged_plan_bytes")) return 0;
  dkv_paged_plan p{};
  layout_of(*batch, p);
  return 4ll * p.words;
}

int dkv_paged_plan_write(const dkv_paged_batch* batch, void* buffer, int64_t bytes, dkv_paged_plan* plan) {
  clear_error();
  if (!batch || !buffer || !plan || ((uintptr_t)buffer & 15)) {
    set_error("dkv_paged_plan_write: null or misaligned pointer argument");
    return DKV_EINVAL;
  }
  if (int rc = check_plan(*batch, "dkv_paged_plan_write")) return rc;
  const int64_t need = dkv_paged_plan_bytes(batch);
  if (bytes < need) {
    set_error("dkv_paged_plan_write: a plan of %lld bytes needed, room for %lld", (long long)need, (long long)bytes);
    return DKV_EINVAL;
  }
  try {
    dkv_paged_plan p{};
    if (int rc = write_plan(*batch, static_cast<int32_t*>(buffer), p)) return rc;
    *plan = p;
    return 0;
  } catch (const std::exception&) {
    set_error("dkv_paged_plan_write: out of host memory");
    return DKV_EINVAL;
  }
}

int dkv_paged_append(const dkv_paged_args* args, void* stream) {
  clear_error();
  if (!args) {
    set_error("dkv_paged_append: null args");
    return DKV_EINVAL;
  }
  if (int rc = check_args(*args, false, "dkv_paged_append")) return rc;
  const dkv_paged_plan& p = args->plan;
  hipLaunchKernelGGL(append_kernel, dim3(2 * (args->bounds ? p.max_items : p.items), (2 * p.heads + 3) / 4), dim3(256), 0, (hipStream_t)stream,
                     *args);
  return (int)hipGetLastError();
}

int dkv_paged_rope_append(const dkv_paged_args* args, const void* qkv, int64_t qkv_row_stride, const void* cos, const void* sin,
                          int64_t cs_row_stride, void* stream) {
  clear_error();
  if (!args) {
    set_error("dkv_paged_rope_append: null args");
    return DKV_EINVAL;
  }
  const dkv_paged_args& a = *args;
  if (int rc = check_args(a, false, "dkv_paged_rope_append")) return rc;
  auto bad = [](const void* x) { return !x || ((uintptr_t)x & 15); };
  if (bad(a.q) || bad(qkv) || bad(cos) || bad(sin) || (a.q_head_stride & 7) || (a.q_tok_stride & 7) || (qkv_row_stride & 7) || (cs_row_stride & 7)) {
    set_error("dkv_paged_rope_append: q, qkv, cos and sin must be 16-byte aligned with strides that are multiples of 8 elements");
    return DKV_EINVAL;
  }
  const dkv_paged_plan& p = a.plan;
  if ((int64_t)p.q_heads + 2 * p.heads > 4 * 65535) {
    set_error("dkv_paged_rope_append: %d query heads are too many", p.q_heads);
    return DKV_EINVAL;
  }
  hipLaunchKernelGGL(rope_append_kernel, dim3(a.bounds ? p.max_items : p.items, (p.q_heads + 2 * p.heads + 3) / 4), dim3(256), 0,
                     (hipStream_t)stream, a, static_cast<const uint16_t*>(qkv), qkv_row_stride, static_cast<const uint16_t*>(cos),
                     static_cast<const uint16_t*>(sin), cs_row_stride);
  return (int)hipGetLastError();
}

int dkv_paged_read(const void* arena, int64_t arena_bytes, const dkv_page_rows* items, int32_t n_items, int32_t layer0,
                   int32_t n_layers, int32_t layers, int32_t heads, void* out, int32_t n_tokens, int32_t out_dtype, void* stream) {
  clear_error();
  if (n_items < 0 || n_tokens < 0 || layer0 < 0 || n_layers <= 0 || (int64_t)layer0 + n_layers > layers || heads <= 0 ||
      (int64_t)layers * heads > 65535 / 2 || out_dtype < 0 || out_dtype > 1) {
    set_error("dkv_paged_read: bad shape (items %d, tokens %d, layers [%d, %d + %d) of %d, heads %d)", n_items, n_tokens, layer0, layer0,
              n_layers, layers, heads);
    return DKV_EINVAL;
  }
  if (n_items == 0) return 0;
  if (!arena || !items || !out || ((uintptr_t)arena & 15) || ((uintptr_t)out & 15)) {
    set_error("dkv_paged_read: null or misaligned pointer argument");
    return DKV_EINVAL;
  }
  const int64_t grains = arena_bytes / grain_bytes(layers, heads);
  for (int i = 0; i < n_items; ++i) {
    const dkv_page_rows& r = items[i];
    if ((r.page & 3) > 2 || (int64_t)(r.page >> 2) + page_grains(page_bits(r.page)) > grains || r.row0 < 0 || r.rows <= 0 ||
        r.row0 > TILE - r.rows || r.token < 0 || r.token > n_tokens - r.rows) {
      set_error("dkv_paged_read: item %d (page %u, rows [%d, %d + %d), token %d) lies outside the arena, its page or the output", i,
                r.page, r.row0, r.row0, r.rows, r.token);
      return DKV_EINVAL;
    }
  }
  for (int i = 0; i < n_items; i += ARG_ITEMS) {
    const int n = std::min(ARG_ITEMS, n_items - i);
    Items block{};
    memcpy(block.at, items + i, n * sizeof(dkv_page_rows));
    hipLaunchKernelGGL(read_kernel, dim3(n, (2 * heads * n_layers + 3) / 4), dim3(256), 0, (hipStream_t)stream, block,
                       static_cast<const uint8_t*>(arena), layer0, n_layers, layers, heads, out, (int64_t)n_tokens, out_dtype);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  return 0;
}

int dkv_paged_move(const void* src, int64_t src_bytes, void* dst, int64_t dst_bytes, const dkv_page_move* moves, int32_t n_moves,
                   int32_t layers, int32_t heads, void* stream) {
  clear_error();
  if (n_moves < 0 || layers <= 0 || heads <= 0 || (int64_t)layers * heads > 65535 / 2) {
    set_error("dkv_paged_move: bad shape (moves %d, layers %d, heads %d)", n_moves, layers, heads);
    return DKV_EINVAL;
  }
  if (n_moves == 0) return 0;
  if (!src || !dst || !moves || ((uintptr_t)src & 15) || ((uintptr_t)dst & 15)) {
    set_error("dkv_paged_move: null or misaligned pointer argument");
    return DKV_EINVAL;
  }
  struct Span {  // tiles that are read (or pages that are written) by a move
    int64_t at, end;
    int row, rows;
    bool write;
  };
  try {
    std::vector<Span> spans;
    for (int i = 0; i < n_moves; ++i) {
      const dkv_page_move& m = moves[i];
      const int64_t from = slab_bytes(m.src_rows, m.bits, layers, heads), to = slab_bytes(TILE, m.bits, layers, heads);
      if ((m.bits != 4 && m.bits != 8 && m.bits != 16) || m.rows < 1 || m.src_rows > TILE || m.src_row + m.rows > m.src_rows ||
          m.dst_row + m.rows > TILE || m.src_offset < 0 || (m.src_offset & 15) || m.src_offset > src_bytes - from || m.dst_offset < 0 ||
          (m.dst_offset & 15) || m.dst_offset > dst_bytes - to) {
        set_error("dkv_paged_move: move %d (%d bits, rows [%d, +%d) of %d at byte %lld to row %d at %lld) lies outside an arena or tile", i,
                  m.bits, m.src_row, m.rows, m.src_rows, (long long)m.src_offset, m.dst_row, (long long)m.dst_offset);
        return DKV_EINVAL;
      }
      spans.push_back(Span{m.dst_offset, m.dst_offset + to, m.dst_row, m.rows, true});
      if (src == dst) spans.push_back(Span{m.src_offset, m.src_offset + from, m.src_row, m.rows, false});
    }
    // Sorted by place, spans of one page follow each other: two of them may meet only in rows that neither shares, or where both read.
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.at != b.at ? a.at < b.at : a.row < b.row; });
    int64_t reach = -1, reach_write = -1;  // ends of the spans before, of those that write
    for (size_t i = 0, j; i < spans.size(); i = j) {
      bool writes = false, clash = false;
      int rows_end = 0, write_end = 0;
      int64_t end = spans[i].end;
      for (j = i; j < spans.size() && spans[j].at == spans[i].at; ++j) {
        const Span& s = spans[j];
        clash = clash || s.end != spans[i].end || s.row < (s.write ? rows_end : write_end);
        rows_end = std::max(rows_end, s.row + s.rows);
        if (s.write) writes = true, write_end = std::max(write_end, s.row + s.rows);
        end = std::max(end, s.end);
      }
      if (clash || spans[i].at < (writes ? reach : reach_write)) {
        set_error("dkv_paged_move: the moves write rows (at byte %lld) that they also read or write elsewhere", (long long)spans[i].at);
        return DKV_EINVAL;
      }
      reach = std::max(reach, end);
      if (writes) reach_write = std::max(reach_write, end);
    }
  } catch (const std::exception&) {
    set_error("dkv_paged_move: out of host memory");
    return DKV_EINVAL;
  }
  return launch_moves(src, dst, moves, n_moves, layers, heads, stream);
}

}  // extern "C"
