// Eviction (gfx950): a cache's packed rows, less the tokens of the smallest attention mass, into another arena.
//
// The segments between the protected ends become one segment a width. Every layer and KV head keeps its own rows of
// each width, as many as the host says, so the tile table is known before the kernels run and nothing waits for the
// device: history rows carry no mask and no position of their own, so a tile may hold other tokens in every head.
// Three launches: where each token lies and which tokens each width has, with the new tile table; the choice, a radix
// search for the smallest kept mass per (layer, head, width); and the move, each kept row read and written
// once.
// Measured (kernel times): 65531 to 16384 tokens, 4 layers of 8 heads: 9.0 + 31.8 (96 workgroups: three radix steps and
// their barriers over up to 26000 keys each) + 51.5 us (148 MB read and written, 2.9 TB/s where a large copy reaches 5.2: a
// row is 32 to 128 bytes at an address of its own). 8128 to 4096, 8 layers of 5: 6.2 + 12.2 + 11.1; a call's host part, some 60 us, is longer.
#include "dkv_select.h"

namespace dkv {
namespace evict {

constexpr int THREADS = 1024;  // of a choosing workgroup

__device__ __forceinline__ int class_of(const dkv_evict_args& e, int bits) {
  for (int c = 0; c < e.n_classes; ++c)
    if (e.class_bits[c] == bits) return c;
  return 3;  // no token of this width stays
}

// The middle's tokens kept before class c, and their tiles.
__host__ __device__ inline int rows_before(const dkv_evict_args& e, int c) {
  int n = 0;
  for (int i = 0; i < c; ++i) n += e.class_keep[i];
  return n;
}
__host__ __device__ inline int tiles_before(const dkv_evict_args& e, int c) {
  int n = 0;
  for (int i = 0; i < c; ++i) n += (e.class_keep[i] + TILE - 1) / TILE;
  return n;
}
__host__ __device__ inline int64_t bytes_before(const dkv_evict_args& e, int c) {
  int64_t n = 0;
  for (int i = 0; i < c; ++i) n = segment_end(n, e.class_keep[i], e.class_bits[i], e.layers, e.heads);
  return n;
}

// The middle's tokens: place[token - lead_tokens] is its tile, and order lists a class's tokens after another's.
struct Work {
  int32_t* place;
  int32_t* order;
};
__host__ __device__ inline int held_before(const dkv_evict_args& e, int c) {
  int n = 0;
  for (int i = 0; i < c; ++i) n += e.class_held[i];
  return n;
}

constexpr int MAP_TILES = 128;  // of the middle, a workgroup

// Rows of each class, in 21 bits each.
__device__ __forceinline__ uint64_t rows_by_class(const dkv_evict_args& e, const dkv_tile& t) {
  const int c = class_of(e, t.bits);
  return c < 3 ? (uint64_t)t.rows << (21 * c) : 0;
}

__global__ __launch_bounds__(THREADS) void map_kernel(dkv_evict_args e, Work w) {
  __shared__ int before[3], at[MAP_TILES], start[MAP_TILES], rows[MAP_TILES];
  __shared__ uint64_t half;
  const int i = blockIdx.x * THREADS + threadIdx.x, mid_tiles = tiles_before(e, e.n_classes);
  const int tail_tiles = e.n_tiles - e.end_tile;
  if (i < e.lead_tiles) {
    e.out_tiles[i] = e.tiles[i];
  } else if (i < e.lead_tiles + mid_tiles) {
    int c = e.n_classes - 1, t = i - e.lead_tiles;
    while (t < tiles_before(e, c)) --c;
    t -= tiles_before(e, c);
    dkv_tile d;
    d.offset = e.lead_bytes + bytes_before(e, c) + t * slab_bytes(TILE, e.class_bits[c], e.layers, e.heads);
    d.token_start = e.lead_tokens + rows_before(e, c) + t * TILE;
    d.rows = (uint16_t)min(TILE, e.class_keep[c] - t * TILE);
    d.bits = (uint8_t)e.class_bits[c];
    d.reserved = 0;
    e.out_tiles[i] = d;
  } else if (i < e.lead_tiles + mid_tiles + tail_tiles) {
    dkv_tile d = e.tiles[e.end_tile + i - e.lead_tiles - mid_tiles];
    d.offset += e.lead_bytes + bytes_before(e, e.n_classes) - e.tail_offset;
    d.token_start += e.lead_tokens + rows_before(e, e.n_classes) - e.end_token;
    e.out_tiles[i] = d;
  }
  const int first = e.lead_tiles + blockIdx.x * MAP_TILES, last = min(e.end_tile, first + MAP_TILES);
  if (first >= last) return;
  // rows of each class in the middle's tiles before these
  if (threadIdx.x < 3) before[threadIdx.x] = 0;
  __syncthreads();
  int mine[3] = {0, 0, 0};
  for (int t = e.lead_tiles + threadIdx.x; t < first; t += THREADS) {
    const dkv_tile d = e.tiles[t];
    const int c = class_of(e, d.bits);
#pragma unroll
    for (int j = 0; j < 3; ++j) mine[j] += c == j ? d.rows : 0;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (mine[j]) atomicAdd(&before[j], mine[j]);
  // and in these, before each: two waves scan them
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = first + threadIdx.x;
  dkv_tile d = {};
  uint64_t upto = 0;
  if (wave < MAP_TILES / 64) {
    if (t < last) d = e.tiles[t];
    upto = t < last ? rows_by_class(e, d) : 0;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint64_t o = (uint64_t)(uint32_t)__shfl_up((int)upto, k, 64) | (uint64_t)(uint32_t)__shfl_up((int)(upto >> 32), k, 64) << 32;
      if (lane >= k) upto += o;
    }
    if (threadIdx.x == 63) half = upto;
  }
  __syncthreads();
  if (wave < MAP_TILES / 64 && t < last) {
    start[threadIdx.x] = d.token_start - e.lead_tokens, rows[threadIdx.x] = d.rows;
    if (wave == 1) upto += half;
    const int c = class_of(e, d.bits);
    at[threadIdx.x] = c < 3 ? held_before(e, c) + before[c] + (int)(upto >> (21 * c) & ((1 << 21) - 1)) - d.rows : -1;
  }
  __syncthreads();
  for (int k = wave; k < last - first; k += THREADS / 64) {
    if (lane >= rows[k]) continue;
    const int token = start[k] + lane;
    w.place[token] = first + k;
    if (at[k] >= 0) w.order[at[k] + lane] = token;
  }
}

// blockIdx: (layer * heads + head, class). The class's tokens of the largest masses, in token order; equal masses
// keep the earlier token. Class 0 also lists the protected ends. Up to N * THREADS keys stay in registers: 65531 to 16384
// tokens, read back, 146 us with N = 32 and 164 with keys loaded again each time (N = 0); 8128 to 4096 124 with N = 4, 128.
template <int N>
__global__ __launch_bounds__(THREADS) void choose_kernel(dkv_evict_args e, Work w) {
  __shared__ SelectScratch<THREADS, 11> scratch;
  const int lh = blockIdx.x, c = blockIdx.y;
  const int mid = rows_before(e, e.n_classes), tail = e.tokens - e.end_token;
  const float* mass = e.mass + lh * e.mass_stride;
  int32_t* kept = e.kept + (int64_t)lh * (e.lead_tokens + mid + tail);
  float* out = e.out_mass + lh * e.out_mass_stride;
  if (c == 0) {
    for (int i = threadIdx.x; i < e.lead_tokens; i += THREADS) kept[i] = i, out[i] = mass[i];
    for (int i = threadIdx.x; i < tail; i += THREADS)
      kept[e.lead_tokens + mid + i] = e.end_token + i, out[e.lead_tokens + mid + i] = mass[e.end_token + i];
    for (int64_t i = e.lead_tokens + mid + tail + threadIdx.x; i < e.out_mass_stride; i += THREADS) out[i] = 0.f;
  }
  if (c >= e.n_classes) return;
  mass += e.lead_tokens;
  const int32_t* order = w.order + held_before(e, c);
  auto key = [&](int i) { return max(order_key(mass[order[i]]), 1u); };  // (1: not a number, below every number)
  const int first = e.lead_tokens + rows_before(e, c), keep = e.class_keep[c];
  Elements<THREADS, N, decltype(key)>(e.class_held[c], key).largest(scratch, (uint32_t)keep, [&](int to, int i) {
    kept[first + to] = i;
  });
  __syncthreads();
  // Places become tokens, where they lie. Loads are in flight together; a thread with fewer than AHEAD reads its own first
  // place again, never another thread's, which may hold a token by then: an index past the class.
  constexpr int AHEAD = 8;
  for (int i0 = threadIdx.x; i0 < keep; i0 += AHEAD * THREADS) {
    int token[AHEAD];
    float m[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) token[j] = kept[first + (i0 + j * THREADS < keep ? i0 + j * THREADS : i0)];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) token[j] = order[token[j]];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) m[j] = mass[token[j]];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (const int i = i0 + j * THREADS; i < keep) kept[first + i] = e.lead_tokens + token[j], out[first + i] = m[j];
  }
}

// One row's 16-byte pieces: 2, 4 or 8 lanes. The rows of K and V of a (new tile, layer, head) move in one wave: lane
// r first finds where row r lies, then the lanes of a row take its address from it.
template <int BITS>
__device__ __forceinline__ void move_rows(const dkv_evict_args& e, const dkv_tile& d, int layer, int h, const int32_t* kept,
                                          const int32_t* place, int lane) {
  constexpr int PIECES = BITS / 2, ROWS = 64 / PIECES, STEPS = TILE / ROWS;  // rows an instruction, instructions a tile
  const int token = kept[min(lane, d.rows - 1)];
  const dkv_tile from = e.tiles[place[token - e.lead_tokens]];
  const int row = token - from.token_start;
  const int64_t from_sb = subblock_bytes(from.rows, BITS), to_sb = subblock_bytes(d.rows, BITS);
  const int64_t block = (int64_t)(layer * 2) * e.heads + h;
  const uint8_t* src = static_cast<const uint8_t*>(e.arena) + from.offset + block * from_sb;
  uint8_t* dst = static_cast<uint8_t*>(e.out_arena) + d.offset + block * to_sb;
  const uint64_t k_row = (uint64_t)(src + (int64_t)row * (8 * BITS)), v_gap = (uint64_t)(e.heads * from_sb);
  u32x4 x[2][STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int r = min(s * ROWS + lane / PIECES, d.rows - 1);
    const uint64_t at = (uint64_t)(uint32_t)__shfl((int)k_row, r, 64) | (uint64_t)(uint32_t)__shfl((int)(k_row >> 32), r, 64) << 32;
    const uint64_t gap = (uint64_t)(uint32_t)__shfl((int)v_gap, r, 64) | (uint64_t)(uint32_t)__shfl((int)(v_gap >> 32), r, 64) << 32;
    x[0][s] = *reinterpret_cast<const u32x4*>(at + lane % PIECES * 16);
    x[1][s] = *reinterpret_cast<const u32x4*>(at + gap + lane % PIECES * 16);
  }
  float2 as[2];
  if (BITS < 16) {
    const uint8_t* meta = src + (int64_t)from.rows * (8 * BITS) + 8 * row;
    as[0] = *reinterpret_cast<const float2*>(meta);
    as[1] = *reinterpret_cast<const float2*>(meta + v_gap);
  }
  const int64_t to_gap = e.heads * to_sb;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      if (s * ROWS + lane / PIECES < d.rows) *reinterpret_cast<u32x4*>(dst + kv * to_gap + (s * 64 + lane) * 16) = x[kv][s];
    if (BITS < 16 && lane < d.rows)
      *reinterpret_cast<float2*>(dst + kv * to_gap + (int64_t)d.rows * (8 * BITS) + 8 * lane) = as[kv];
  }
}

constexpr int COPY_BYTES = 32768;  // of a copying workgroup

// Workgroups [0, gathers): four (layer, head) of a new tile of the middle, a wave each; the rest copy the ends.
__global__ __launch_bounds__(256) void move_kernel(dkv_evict_args e, int gathers, const int32_t* place) {
  const int lhs = e.layers * e.heads, per_tile = (lhs + 3) / 4;
  if ((int)blockIdx.x < gathers) {
    const int lh = blockIdx.x % per_tile * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (lh >= lhs) return;
    const dkv_tile d = e.out_tiles[e.lead_tiles + blockIdx.x / per_tile];
    const int total = e.lead_tokens + rows_before(e, e.n_classes) + e.tokens - e.end_token;
    const int32_t* kept = e.kept + (int64_t)lh * total + d.token_start;
    const int bits = __builtin_amdgcn_readfirstlane((int)d.bits);
    if (bits == 4) move_rows<4>(e, d, lh / e.heads, lh % e.heads, kept, place, lane);
    else if (bits == 8) move_rows<8>(e, d, lh / e.heads, lh % e.heads, kept, place, lane);
    else move_rows<16>(e, d, lh / e.heads, lh % e.heads, kept, place, lane);
    return;
  }
  // 16-byte pieces of the leading tiles, which stay where they were, then of the trailing ones
  const int64_t pieces = (e.lead_bytes + e.tail_bytes) / 16, lead = e.lead_bytes / 16;
  const u32x4* from = static_cast<const u32x4*>(e.arena);
  u32x4* to = static_cast<u32x4*>(e.out_arena);
  const int64_t tail_from = e.tail_offset / 16 - lead, tail_to = bytes_before(e, e.n_classes) / 16;
  const int64_t first = (int64_t)(blockIdx.x - gathers) * (COPY_BYTES / 16);
#pragma unroll
  for (int i = 0; i < COPY_BYTES / 16 / 256; ++i) {
    const int64_t p = first + i * 256 + threadIdx.x;
    if (p < pieces) to[p < lead ? p : p + tail_to] = from[p < lead ? p : p + tail_from];
  }
}

static bool fits(const dkv_evict_args& e) {
  if (e.layers <= 0 || e.heads <= 0 || (int64_t)e.layers * e.heads > INT32_MAX / 4 || e.n_tiles < 0 || e.lead_tiles < 0 ||
      e.end_tile < e.lead_tiles || e.n_tiles < e.end_tile || e.lead_tokens < 0 || e.end_token < e.lead_tokens ||
      e.tokens < e.end_token || e.n_classes < 0 || e.n_classes > 3 || e.lead_bytes < 0 || e.tail_offset < e.lead_bytes ||
      e.tail_bytes < 0 || (e.lead_bytes & 15) || (e.tail_offset & 15) || (e.tail_bytes & 15))
    return false;
  int64_t kept = 0, held = 0;
  for (int c = 0; c < e.n_classes; ++c) {
    if ((e.class_bits[c] != 4 && e.class_bits[c] != 8 && e.class_bits[c] != 16) || e.class_keep[c] <= 0) return false;
    for (int i = 0; i < c; ++i)
      if (e.class_bits[i] == e.class_bits[c]) return false;
    kept += e.class_keep[c], held += e.class_held[c];
    if (e.class_held[c] < e.class_keep[c]) return false;
  }
  const int64_t total = e.lead_tokens + kept + e.tokens - e.end_token;
  return held <= e.end_token - e.lead_tokens && e.mass_stride >= e.tokens && e.out_mass_stride >= total &&
         e.out_arena_bytes >= e.lead_bytes + bytes_before(e, e.n_classes) + e.tail_bytes &&
         e.arena_bytes >= e.tail_offset + e.tail_bytes;
}

}  // namespace evict
}  // namespace dkv

using namespace dkv;

extern "C" {

int64_t dkv_evict_workspace_bytes(const dkv_evict_args* args) {
  if (!args || args->end_token <= args->lead_tokens) return 0;
  return 8 * ((int64_t)args->end_token - args->lead_tokens);
}

int dkv_evict(const dkv_evict_args* args, void* stream) {
  clear_error();
  if (!args) {
    set_error("dkv_evict: null args");
    return DKV_EINVAL;
  }
  const dkv_evict_args& e = *args;
  if (!evict::fits(e)) {
    set_error("dkv_evict: bad ranges (tiles %d | %d | %d, tokens %d | %d | %d, widths %d, or rows or arenas too small)",
              e.lead_tiles, e.end_tile, e.n_tiles, e.lead_tokens, e.end_token, e.tokens, e.n_classes);
    return DKV_EINVAL;
  }
  if (e.n_tiles == 0) return 0;
  if (!e.arena || !e.tiles || !e.mass || !e.out_arena || !e.out_tiles || !e.out_mass || !e.kept ||
      ((uintptr_t)e.arena & 15) || ((uintptr_t)e.out_arena & 15)) {
    set_error("dkv_evict: null or misaligned pointer argument");
    return DKV_EINVAL;
  }
  const uint8_t *from = static_cast<const uint8_t*>(e.arena), *to = static_cast<const uint8_t*>(e.out_arena);
  if ((from < to + e.out_arena_bytes && to < from + e.arena_bytes) || e.tiles == e.out_tiles || e.mass == e.out_mass) {
    set_error("dkv_evict: the new arena, tiles and masses must not be the old ones");
    return DKV_EINVAL;
  }
  if (e.workspace_bytes < dkv_evict_workspace_bytes(args) || (!e.workspace && dkv_evict_workspace_bytes(args))) {
    set_error("dkv_evict: workspace of %lld bytes needed, %lld given", (long long)dkv_evict_workspace_bytes(args),
              (long long)e.workspace_bytes);
    return DKV_EINVAL;
  }
  const evict::Work w{static_cast<int32_t*>(e.workspace), static_cast<int32_t*>(e.workspace) + (e.end_token - e.lead_tokens)};
  const int mid_tiles = evict::tiles_before(e, e.n_classes), out_tiles = e.lead_tiles + mid_tiles + e.n_tiles - e.end_tile;
  const int by_tile = (out_tiles + evict::THREADS - 1) / evict::THREADS, lhs = e.layers * e.heads;
  const int by_range = (e.end_tile - e.lead_tiles + evict::MAP_TILES - 1) / evict::MAP_TILES;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(evict::map_kernel, dim3(by_tile > by_range ? by_tile : by_range), dim3(evict::THREADS), 0, st, e, w);
  int n = 0;
  for (int c = 0; c < e.n_classes; ++c) n = e.class_held[c] > n ? e.class_held[c] : n;
  const auto choose = n <= 4 * evict::THREADS    ? evict::choose_kernel<4>
                      : n <= 12 * evict::THREADS ? evict::choose_kernel<12>
                      : n <= 32 * evict::THREADS ? evict::choose_kernel<32>
                                                 : evict::choose_kernel<0>;
  hipLaunchKernelGGL(choose, dim3(lhs, e.n_classes ? e.n_classes : 1), dim3(evict::THREADS), 0, st, e, w);
  const int64_t gathers = (int64_t)mid_tiles * ((lhs + 3) / 4);
  const int64_t copies = (e.lead_bytes + e.tail_bytes + evict::COPY_BYTES - 1) / evict::COPY_BYTES;
  if (gathers + copies > INT32_MAX) {
    set_error("dkv_evict: too many rows for one call");
    return DKV_EINVAL;
  }
  if (gathers + copies)
    hipLaunchKernelGGL(evict::move_kernel, dim3((unsigned)(gathers + copies)), dim3(256), 0, st, e, (int)gathers, w.place);
  return (int)hipGetLastError();
}

}  // extern "C"
