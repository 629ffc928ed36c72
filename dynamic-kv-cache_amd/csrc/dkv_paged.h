// Paged caches (dkv_paged.hip: plans, pack, read, move; dkv_paged_attn.hip, dkv_paged_short.h, dkv_paged_prompt.hip: attention): the
// page layout, and what a step's plan holds in device memory.
#pragma once
#include "dkv_common.h"

namespace dkv {
namespace paged {

constexpr int GRAIN_ROW = 512;  // bytes of a sub-block in one grain: 2560, 4608 and 8192 are multiples of it

__host__ __device__ inline int page_bits(uint32_t page) { return 4 << (page & 3); }
__host__ __device__ inline int page_sub(int bits) { return 512 * bits + (bits < 16 ? 512 : 0); }  // subblock_bytes(64, bits)
__host__ __device__ inline int64_t grain_bytes(int layers, int heads) { return (int64_t)GRAIN_ROW * 2 * layers * heads; }
__host__ __device__ inline int page_grains(int bits) { return page_sub(bits) / GRAIN_ROW; }

// The K sub-block of (layer, head) of a page; V's lies heads sub-blocks behind it.
__device__ __forceinline__ int64_t page_at(uint32_t page, int layer, int layers, int heads, int h) {
  return (int64_t)(page >> 2) * grain_bytes(layers, heads) + ((int64_t)layer * 2 * heads + h) * page_sub(page_bits(page));
}

// A plan's first words: how many records of each kind it has.
enum { N_ITEMS, N_WORK, N_LONG, N_MERGES, HEAD_WORDS = 16 };

// Rows of the step that go into one page: dkv_page_rows. History pages: {page, rows of it that are history}.
struct Page {
  uint32_t page;
  int32_t rows;
};

// One workgroup's share of a sequence's (or, over pages that several sequences have in common, a group's) attention, for
// each KV head: units [u0, u1) for block `block` of its query rows. Unit u is page first_page + u of the plan while u is
// below n_pages (at 4 bits below n4, 8 below n8, else 16: attention takes keys in any order), then 64 new tokens each. Query
// row r is token r / G, query head r % G of the KV head; `count` tokens from token0 of the step on. The block's rows go to the
// partial rows from `part` on, or where that is negative to the output.
struct Work {
  int32_t first_page, n4, n8, n_pages, token0, count, block, u0, u1, part, reserved[2];
};

// Query rows [row0, row0 + 16) of a sequence that has `rows` of them from token0 on, joined from its own partials (row
// row0 at part, the splits `stride` rows apart) and those of its group (shared, shared_stride). splits: its own, and the
// group's in the upper half.
struct Merge {
  int32_t token0, rows, row0, part, stride, shared, shared_stride;
  uint32_t splits;
};

// A record of a plan, or a part of one, by scalar loads: no launch writes the plan that it reads.
template <class T>
__device__ __forceinline__ T plan_record(const int32_t* plan, int at, int i) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  const scalar_ptr from = (scalar_ptr)(plan + at + i * (int)(sizeof(T) / 4));
  union {
    T t;
    int32_t w[sizeof(T) / 4];
  } x;
#pragma unroll
  for (int j = 0; j < (int)(sizeof(T) / 4); ++j) x.w[j] = from[j];
  return x.t;
}

constexpr int SHORT_BLOCK = 16;  // query rows of a block of the kernel for few rows (dkv_paged_short.h)
constexpr int LONG_BLOCK = 256;  // of the one for many (dkv_paged_prompt.hip)

// Four elements of an output row.
__device__ __forceinline__ void store4(void* out, int out_dtype, int64_t at, float __attribute__((ext_vector_type(4))) x) {
  if (out_dtype == 1)
    *reinterpret_cast<float __attribute__((ext_vector_type(4)))*>(static_cast<float*>(out) + at) = x;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

__device__ __forceinline__ bool bad_bf16(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }  // infinite or NaN

// The launch of many query rows, with workgroups of few ones behind it.
void launch_long(const dkv_paged_args& a, int n_long, int n_short, float* part_o, float2* part_ml, hipStream_t s);

int check_args(const dkv_paged_args& a, bool attend, const char* what);

// The launches of moves that are known to be in place (dkv_paged_move checks its own). A null dst moves nothing.
int launch_moves(const void* src, void* dst, const dkv_page_move* moves, int n, int layers, int heads, void* stream);

}  // namespace paged
}  // namespace dkv
