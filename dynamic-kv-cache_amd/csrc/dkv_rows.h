// Packed rows straight into MFMA operands: what the sparse-attention and attention-mass kernels share.
//
// S^T = K Q^T and O^T = V^T P^T as v_mfma_f32_16x16x32_bf16, a wave per 64-key unit, keys on M of the
// first product, query rows on N of both. With lane l = 16 g + c:
//   - K: lane (c, g) holds elements [16 g, 16 g + 16) of key 16 b + c of every 16-key block b: one piece of
//     the packed row (8, 16 or 32 bytes). The dot product runs over the elements in any order, so the two
//     operands of a block are elements 16 g + [0, 8) and 16 g + [8, 16) in K and Q alike;
//   - S^T: lane (c, g) gets query row c and keys 16 b + 4 g + i, which is a P^T operand as it stands (the
//     product over keys runs in any order too): element 4 (b % 2) + i of operand b / 2;
//   - V: lane (c, g) holds elements [4 c, 4 c + 4) of keys 16 b + 4 g + i, so element 4 c + db of those keys
//     is the V^T operand of output block db, without an exchange between lanes;
//   - O^T: lane (c, g) gets query row c, element 16 g + 4 i + db.
// No byte passes through LDS.
#pragma once
#include "dkv_attn_common.h"

namespace dkv {
namespace rows {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

union Op {  // one lane's 8 elements of an MFMA operand
  bf16x8 v;
  uint32_t u[4];
};

__device__ __forceinline__ f32x4 mfma(const Op& a, const Op& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}

// Where a unit's rows are: packed rows of a tile, or the chunk's own bf16 rows (BITS 16) at any stride.
// `rows` rows can be read (1..64); keys outside [low, high) are not visible.
struct UnitRows {
  const uint8_t* k;
  const uint8_t* v;
  uint32_t k_stride, v_stride;  // bytes from row to row, below 2^24: a row's offset is a 24-bit product (a 64-bit one is four slow ones)
  int bits, rows, low, high;
};

__device__ __forceinline__ UnitRows tile_rows(const dkv_attn_args& a, const dkv_tile& t, int past, int h) {
  UnitRows u;
  u.bits = t.bits;
  u.rows = t.rows;
  u.low = 0;
  u.high = min((int)t.rows, past - t.token_start);
  const int64_t sb = subblock_bytes(t.rows, t.bits);
  const uint8_t* base = static_cast<const uint8_t*>(a.arena) + t.offset;
  u.k = base + ((int64_t)(a.layer * 2 + 0) * a.heads + h) * sb;
  u.v = base + ((int64_t)(a.layer * 2 + 1) * a.heads + h) * sb;
  u.k_stride = u.v_stride = row_bytes(t.bits);
  return u;
}

// Chunk rows [64 piece, ...) of KV head h.
__device__ __forceinline__ UnitRows chunk_rows(const dkv_attn_args& a, int piece, int h) {
  UnitRows u;
  const int first = piece * TILE;
  u.bits = 16;
  u.rows = min(TILE, a.nq - first);
  u.low = 0;
  u.high = u.rows;
  u.k = static_cast<const uint8_t*>(a.k_new) + 2 * (h * a.kn_head_stride + first * a.kn_tok_stride);
  u.v = static_cast<const uint8_t*>(a.v_new) + 2 * (h * a.vn_head_stride + first * a.vn_tok_stride);
  u.k_stride = (uint32_t)(2 * a.kn_tok_stride);  // (of a single row, whatever it is)
  u.v_stride = (uint32_t)(2 * a.vn_tok_stride);
  return u;
}

// Value e of a loaded piece: the code as fp32 (BITS 4 and 8).
template <int BITS>
__device__ __forceinline__ float code_at(const uint32_t* w, int e) {
  if (BITS == 8) return (float)((w[e >> 2] >> (8 * (e & 3))) & 0xffu);
  return (float)((w[e >> 3] >> (4 * (e & 7))) & 0xfu);
}

// x as the sum of TERMS bf16 values: two keep all but 2^-17 of a value, three all but 2^-25.
template <int TERMS>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t (&out)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    out[t] = pack_bf16(x0, x1);
    if (t + 1 < TERMS) {
      x0 -= bf16_lo(out[t]);
      x1 -= bf16_hi(out[t]);
    }
  }
}

// At precision 0 a key or value is its fp32 value rounded to bf16, which is what attention multiplies. At precision 1 a
// packed row is taken as it is stored, scale * (code - centre) + (offset + scale * centre): the centred codes are exact
// in bf16, so one MFMA gives their products without a value being unpacked, and scale and offset come after (keys) or go
// into the weights (values). 16-bit rows are bf16 at both.
template <int BITS, int PREC>
constexpr bool AFFINE = PREC == 1 && BITS < 16;
template <int BITS>
constexpr float CENTRE = BITS == 4 ? 8.f : 128.f;

// Codes e and e + 1 (or the elements of a 16-bit row) as a bf16 pair, unpacked as PREC asks.
template <int BITS, int PREC>
__device__ __forceinline__ uint32_t unpack_pair(float c0, float c1, float scale0, float offset0, float scale1, float offset1) {
  if (AFFINE<BITS, PREC>) return pack_bf16(c0 - CENTRE<BITS>, c1 - CENTRE<BITS>);
  return pack_bf16(c0 * scale0 + offset0, c1 * scale1 + offset1);
}

// 16 elements of a key and its (offset, scale), as loaded.
struct KeyPiece {
  uint32_t w[8];
  float2 as;
};

template <int BITS>
__device__ __forceinline__ void load_key(const UnitRows& u, int row, int g, KeyPiece& p) {
  const int r = row < u.rows ? row : 0;
  const uint8_t* at = u.k + (__umul24(r, u.k_stride) + g * 2 * BITS);
  if (BITS == 4) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(at);
    p.w[0] = x[0], p.w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < BITS / 8; ++i) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(at + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) p.w[4 * i + j] = x[j];
    }
  }
  if (BITS < 16) p.as = *reinterpret_cast<const float2*>(u.k + (u.rows * (8 * BITS) + 8 * r));
}

// The operands of a key: elements 16 g + 8 half + [0, 8).
template <int BITS, int PREC>
__device__ __forceinline__ void key_ops(const KeyPiece& p, Op (&op)[2]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    op[j / 4].u[j % 4] = BITS == 16 ? p.w[j]
                                    : unpack_pair<BITS, PREC>(code_at<BITS>(p.w, 2 * j), code_at<BITS>(p.w, 2 * j + 1), p.as.y,
                                                              p.as.x, p.as.y, p.as.x);
}

// (offset + scale * centre, scale) of the lane's rows 16 b + 4 g + i of a packed tile: as[b][i / 2][2 (i % 2) + ...].
// Two rows' pairs in one load: a pair whose first row the tile has lies within the sub-block, whose size is rounded up
// to 16 bytes.
template <int BITS>
__device__ __forceinline__ void load_scales(const uint8_t* base, int rows, int g, f32x4 (&as)[4][2]) {
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * b + 4 * g + 2 * i;
      as[b][i] = *reinterpret_cast<const f32x4*>(base + (rows * (8 * BITS) + 8 * (row < rows ? row : 0)));
    }
}

// Products of a query row with a unit's centred codes as scores: scale * product + offset' * (sum of the query).
template <int BITS>
__device__ __forceinline__ void affine_scores(const f32x4 (&as)[4][2], float query_sum, f32x4 (&s)[4]) {
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float offset = as[b][i / 2][2 * (i % 2)], scale = as[b][i / 2][2 * (i % 2) + 1];
      s[b][i] = __builtin_fmaf(scale, s[b][i], __builtin_fmaf(scale, CENTRE<BITS>, offset) * query_sum);
    }
}

// A query row's operands (elements 16 g + [0, 8) and [8, 16)); zeros where there is no row.
__device__ __forceinline__ void query_ops(const uint16_t* row, bool there, int g, Op (&q)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4 x = there ? *reinterpret_cast<const u32x4*>(row + 16 * g + 8 * i) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) q[i].u[j] = x[j];
  }
}

// The sum of a query row's elements, in the four lanes that hold it.
__device__ __forceinline__ float row_sum(float x);
__device__ __forceinline__ float query_sum(const Op (&q)[2]) {
  float x = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) x += bf16_lo(q[i].u[j]) + bf16_hi(q[i].u[j]);
  return row_sum(x);
}

// Elements [4 c, 4 c + 4) of the lane's 16 keys 16 b + 4 g + i of V, as loaded.
template <int BITS>
struct ValuePiece {
  uint32_t w[4][4][BITS == 16 ? 2 : 1];
};

template <int BITS>
__device__ __forceinline__ void load_values(const UnitRows& u, int c, int g, ValuePiece<BITS>& p) {
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * b + 4 * g + i, r = row < u.rows ? row : 0;
      const uint8_t* at = u.v + __umul24(r, u.v_stride);
      if (BITS == 4) {
        p.w[b][i][0] = *reinterpret_cast<const uint16_t*>(at + 2 * c);
      } else if (BITS == 8) {
        p.w[b][i][0] = *reinterpret_cast<const uint32_t*>(at + 4 * c);
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(at + 8 * c);
        p.w[b][i][0] = x[0];
        p.w[b][i][1 % (BITS == 16 ? 2 : 1)] = x[1];
      }
    }
}

// The operands of output block db: keys 16 (2 step + j / 4) + 4 g + j % 4.
template <int BITS, int PREC>
__device__ __forceinline__ void value_ops(const ValuePiece<BITS>& p, const f32x4 (&as)[4][2], int db, Op (&op)[2]) {
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      uint32_t t;
      if (BITS == 16) {
        const uint32_t x0 = p.w[b][i][(db >> 1) % (BITS == 16 ? 2 : 1)], x1 = p.w[b][i + 1][(db >> 1) % (BITS == 16 ? 2 : 1)];
        t = db & 1 ? (x0 >> 16) | (x1 & 0xffff0000u) : (x0 & 0xffffu) | (x1 << 16);
      } else {
        const f32x4 m = as[b][i / 2];
        t = unpack_pair<BITS, PREC>(code_at<BITS>(p.w[b][i], db), code_at<BITS>(p.w[b][i + 1], db), m[1], m[0], m[3], m[2]);
      }
      op[b / 2].u[2 * (b % 2) + i / 2] = t;
    }
}

// Max / sum over the four lanes that hold one query row (c, c + 16, c + 32, c + 48).
__device__ __forceinline__ float row_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = max_nn(__uint_as_float(r[0]), __uint_as_float(r[1]));
  auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_nn(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float row_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

}  // namespace rows
}  // namespace dkv
