// The pages of a paged cache and the sequences that hold them: host bookkeeping, and the launches that move rows.
//
// The arena is cut into blocks of 48 grains that hold pages of one width while they hold any: 9, 5 or 3 pages of 4, 8 or
// 16 bits, of which 45, 45 or 48 grains are used. So no free room is too small for any page but within a block, and the
// pages of a width can be brought together into as few blocks as hold them, in one round of moves: every move goes from
// a block that is emptied to a free place of one that stays. A sequence's last page, unless it is full, is held by that
// sequence alone; the others may be held by several.
#include "dkv_paged.h"
#include <stdio.h>
#include <algorithm>
#include <initializer_list>
#include <map>
#include <mutex>
#include <new>
#include <set>
#include <vector>

namespace dkv {
namespace paged {

constexpr int BLOCK = 48;                        // grains
constexpr int PER_BLOCK[3] = {9, 5, 3};          // pages, by code
constexpr int64_t MOST_BLOCKS = (1 << 30) / BLOCK - 1;  // (a page word has 30 bits for the grain)

struct Sequence {
  std::vector<uint32_t> pages;
  std::vector<int32_t> rows;  // tokens of each page
  int64_t length = 0, dropped = 0;

  int room(int code) const { return !pages.empty() && (int)(pages.back() & 3) == code ? TILE - rows.back() : 0; }
  int fresh(int64_t n, int code) const {  // pages that n more tokens open
    const int64_t left = n - room(code);
    return left > 0 ? (int)((left + TILE - 1) / TILE) : 0;
  }
};

// Some of the blocks, of which it gives the lowest: bits, of every 64 words whether any has one, and so on up to one word.
// (No call allocates after the start, so none of them can fail between two changes.)
class BlockSet {
  std::vector<std::vector<uint64_t>> level;

 public:
  int64_t size = 0;

  explicit BlockSet(int64_t n = 0) {
    do {
      n = (n + 63) / 64;
      level.emplace_back(std::max<int64_t>(n, 1), 0);
    } while (n > 1);
  }
  bool has(int64_t b) const { return level[0][b >> 6] >> (b & 63) & 1; }
  int first() const {
    int64_t b = 0;
    for (size_t i = level.size(); i-- > 0;) b = b << 6 | __builtin_ctzll(level[i][b]);
    return (int)b;
  }
  void insert(int64_t b) {
    if (has(b)) return;
    ++size;
    for (auto& words : level) {
      const bool some = words[b >> 6] != 0;
      words[b >> 6] |= 1ull << (b & 63);
      if (some) return;
      b >>= 6;
    }
  }
  void erase(int64_t b) {
    if (!has(b)) return;
    --size;
    for (auto& words : level) {
      words[b >> 6] &= ~(1ull << (b & 63));
      if (words[b >> 6]) return;
      b >>= 6;
    }
  }
};

}  // namespace paged
}  // namespace dkv

using namespace dkv;
using namespace dkv::paged;

struct dkv_pool {
  int layers, heads, q_heads, precision;
  int64_t grain, blocks;
  std::mutex lock;
  std::vector<int8_t> code;    // of a block's pages, -1: it holds none
  std::vector<uint16_t> used;  // which of its places hold one
  BlockSet empty, part[3];  // blocks without pages; with some and room for more
  int64_t n_pages[3] = {}, n_blocks[3] = {};
  std::vector<int32_t> refs;  // sequences that hold the page at a grain
  std::map<int64_t, Sequence> seqs;
  int64_t next = 0, generation = 0;

  int64_t offset(uint32_t page) const { return (int64_t)(page >> 2) * grain; }
  static uint16_t full(int c) { return (uint16_t)((1 << PER_BLOCK[c]) - 1); }

  uint32_t take(int c) {
    if (!part[c].size) {
      const int b = empty.first();
      part[c].insert(b);
      empty.erase(b);
      code[b] = (int8_t)c;
      ++n_blocks[c];
    }
    const int b = part[c].first(), slot = __builtin_ctz(~(unsigned)used[b]);
    used[b] |= (uint16_t)(1 << slot);
    if (used[b] == full(c)) part[c].erase(b);
    ++n_pages[c];
    const uint32_t g = (uint32_t)b * BLOCK + slot * page_grains(4 << c);
    refs[g] = 1;
    return DKV_PAGE_WORD(g, c);
  }

  void give(uint32_t page) {
    const int c = page & 3, b = (int)((page >> 2) / BLOCK);
    used[b] &= (uint16_t) ~(1 << (page >> 2) % BLOCK / page_grains(4 << c));
    --n_pages[c];
    if (!used[b]) {
      part[c].erase(b);
      code[b] = -1;
      --n_blocks[c];
      empty.insert(b);
    } else {
      part[c].insert(b);
    }
  }

  void release(const uint32_t* pages, size_t n) {  // one holder less of each
    for (size_t i = 0; i < n; ++i)
      if (--refs[pages[i] >> 2] == 0) give(pages[i]);
  }

  // Blocks that hold `need` more pages of each width beside what there is; together: as few as can.
  int64_t blocks_for(const int64_t (&need)[3], bool together) const {
    int64_t n = 0;
    for (int c = 0; c < 3; ++c) {
      const int64_t least = (n_pages[c] + need[c] + PER_BLOCK[c] - 1) / PER_BLOCK[c];
      n += together ? least : std::max(least, n_blocks[c]);
    }
    return n;
  }

  int compact(void* arena, void* stream, int64_t& moved) {
    std::vector<dkv_page_move> moves;
    std::vector<uint32_t> from, to;  // grains
    std::vector<int> held[3];
    for (int b = 0; b < blocks; ++b)
      if (code[b] >= 0) held[code[b]].push_back(b);
    for (int c = 0; c < 3; ++c) {
      auto& h = held[c];
      std::stable_sort(h.begin(), h.end(), [&](int x, int y) { return __builtin_popcount(used[x]) > __builtin_popcount(used[y]); });
      const size_t stay = (size_t)((n_pages[c] + PER_BLOCK[c] - 1) / PER_BLOCK[c]);
      const int size = page_grains(4 << c);
      size_t b = 0;
      int slot = -1;
      for (size_t i = stay; i < h.size(); ++i)
        for (int s = 0; s < PER_BLOCK[c]; ++s) {
          if (!(used[h[i]] >> s & 1)) continue;
          do {  // the next free place of a block that stays
            if (++slot == PER_BLOCK[c]) slot = 0, ++b;
          } while (used[h[b]] >> slot & 1);
          from.push_back((uint32_t)h[i] * BLOCK + s * size), to.push_back((uint32_t)h[b] * BLOCK + slot * size);
          moves.push_back(dkv_page_move{from.back() * grain, to.back() * grain, TILE, 0, 0, TILE, (uint8_t)(4 << c), {}});
        }
    }
    moved = (int64_t)moves.size();
    if (moves.empty()) return 0;
    std::vector<uint32_t> place(refs.size());
    for (size_t g = 0; g < place.size(); ++g) place[g] = (uint32_t)g;
    if (int rc = launch_moves(arena, arena, moves.data(), (int)moves.size(), layers, heads, stream)) return rc;
    for (size_t i = 0; i < from.size(); ++i) place[from[i]] = to[i], refs[to[i]] = refs[from[i]], refs[from[i]] = 0;
    for (auto& s : seqs)
      for (uint32_t& p : s.second.pages) p = place[p >> 2] << 2 | (p & 3);
    for (size_t i = 0; i < to.size(); ++i) {
      const int b = to[i] / BLOCK, c = code[b];
      used[b] |= (uint16_t)(1 << to[i] % BLOCK / page_grains(4 << c));
      if (used[b] == full(c)) part[c].erase(b);
    }
    for (size_t i = 0; i < from.size(); ++i) {
      const int b = from[i] / BLOCK, c = code[b];
      if (c < 0) continue;
      used[b] = 0, code[b] = -1;
      part[c].erase(b), --n_blocks[c], empty.insert(b);
    }
    ++generation;
    return 0;
  }

  // Room for `need` more pages of each width: pages are brought together where that makes it.
  int make_room(const int64_t (&need)[3], void* arena, void* stream, const char* what) {
    if (blocks_for(need, false) <= blocks) return 0;
    if (blocks_for(need, true) > blocks) {
      set_error("%s: paged cache is full: %lld, %lld and %lld new pages at 4, 8 and 16 bits beside %lld, %lld and %lld in %lld blocks", what,
                (long long)need[0], (long long)need[1], (long long)need[2], (long long)n_pages[0], (long long)n_pages[1],
                (long long)n_pages[2], (long long)blocks);
      return DKV_EINVAL;
    }
    int64_t moved;
    return compact(arena, stream, moved);
  }

  Sequence* find(int64_t seq, const char* what) {
    const auto it = seqs.find(seq);
    if (it != seqs.end()) return &it->second;
    set_error("%s: no sequence %lld in this cache", what, (long long)seq);
    return nullptr;
  }

  // Distinct sequences of this cache, or an error.
  int named(const int64_t* ids, int n, std::vector<Sequence*>& out, const char* what) {
    if (n < 0 || (n > 0 && !ids)) {
      set_error("%s: %d sequences, or a null array", what, n);
      return DKV_EINVAL;
    }
    std::set<int64_t> seen;
    for (int i = 0; i < n; ++i) {
      Sequence* s = find(ids[i], what);
      if (!s) return DKV_EINVAL;
      if (!seen.insert(ids[i]).second) {
        set_error("%s: sequence %lld is named twice", what, (long long)ids[i]);
        return DKV_EINVAL;
      }
      out.push_back(s);
    }
    return 0;
  }
};

namespace {

// A call on a pool that needs some pointers beside: its lock, and an error where it throws.
template <class F>
int guarded(dkv_pool* pool, const char* what, std::initializer_list<const void*> needed, F&& f) {
  clear_error();
  if (!pool || std::count(needed.begin(), needed.end(), nullptr)) {
    set_error("%s: null %s", what, pool ? "pointer argument" : "pool");
    return DKV_EINVAL;
  }
  try {
    const std::lock_guard<std::mutex> hold(pool->lock);
    return f(*pool);
  } catch (const std::exception&) {
    set_error("%s: out of host memory", what);
    return DKV_EINVAL;
  }
}

int code_of(int bits) { return bits == 4 ? 0 : bits == 8 ? 1 : bits == 16 ? 2 : -1; }

// What a step asks for: its sequences, widths' codes, new pages by width and the pages of all sequences after it.
struct Ask {
  std::vector<Sequence*> s;
  std::vector<int> code;
  int64_t need[3] = {}, pages = 0;
};

int read_ask(dkv_pool& p, int32_t n, const int64_t* seqs, const int32_t* counts, const int32_t* bits, Ask& a, const char* what) {
  if (n <= 0 || !seqs || !counts || !bits) {
    set_error("%s: no sequences, or a null array", what);
    return DKV_EINVAL;
  }
  if (int rc = p.named(seqs, n, a.s, what)) return rc;
  for (int i = 0; i < n; ++i) {
    const int c = code_of(bits[i]);
    if (c < 0 || counts[i] < 1 || a.s[i]->length + a.s[i]->dropped + counts[i] > INT32_MAX) {
      set_error("%s: %d new tokens at %d bits after %lld", what, counts[i], bits[i], (long long)a.s[i]->length);
      return DKV_EINVAL;
    }
    const int fresh = a.s[i]->fresh(counts[i], c);
    a.code.push_back(c);
    a.need[c] += fresh;
    a.pages += (int64_t)a.s[i]->pages.size() + fresh;
  }
  return 0;
}

}  // namespace

extern "C" {

int dkv_pool_create(int32_t layers, int32_t heads, int32_t q_heads, int32_t precision, int64_t arena_bytes, dkv_pool** pool) {
  clear_error();
  if (!pool || layers <= 0 || heads <= 0 || q_heads <= 0 || q_heads % heads || (int64_t)layers * heads > 65535 / 2 || precision < 0 ||
      precision > 1) {
    set_error("dkv_pool_create: bad shape (%d layers, %d of %d heads) or precision %d", layers, heads, q_heads, precision);
    return DKV_EINVAL;
  }
  const int64_t grain = grain_bytes(layers, heads), blocks = arena_bytes / (grain * BLOCK);
  if (blocks < 1 || blocks > MOST_BLOCKS) {
    set_error("dkv_pool_create: an arena of %lld bytes holds %lld blocks of %lld, not 1 to %lld", (long long)arena_bytes, (long long)blocks,
              (long long)(grain * BLOCK), (long long)MOST_BLOCKS);
    return DKV_EINVAL;
  }
  dkv_pool* p = nullptr;
  try {
    p = new dkv_pool;
    p->layers = layers, p->heads = heads, p->q_heads = q_heads, p->precision = precision, p->grain = grain, p->blocks = blocks;
    p->code.assign(blocks, -1), p->used.assign(blocks, 0), p->refs.assign(blocks * BLOCK, 0);
    p->empty = BlockSet(blocks);
    for (auto& some : p->part) some = BlockSet(blocks);
    for (int b = 0; b < blocks; ++b) p->empty.insert(b);
    *pool = p;
    return 0;
  } catch (const std::exception&) {
    delete p;
    set_error("dkv_pool_create: out of host memory");
    return DKV_EINVAL;
  }
}

int dkv_pool_destroy(dkv_pool* pool) {
  delete pool;
  return 0;
}

int dkv_pool_info_get(dkv_pool* pool, dkv_pool_info* info) {
  return guarded(pool, "dkv_pool_info_get", {info}, [&](dkv_pool& p) {
    *info = dkv_pool_info{p.grain, p.blocks, p.empty.size, (int64_t)p.seqs.size(), p.generation,
                          {p.n_pages[0], p.n_pages[1], p.n_pages[2]}, {p.n_blocks[0], p.n_blocks[1], p.n_blocks[2]}};
    return 0;
  });
}

int dkv_pool_generation(dkv_pool* pool, const int64_t** at) {
  return guarded(pool, "dkv_pool_generation", {at}, [&](dkv_pool& p) {
    *at = &p.generation;
    return 0;
  });
}

int dkv_pool_sequence(dkv_pool* pool, int64_t seq, int64_t* length, int64_t* dropped, int32_t* pages) {
  return guarded(pool, "dkv_pool_sequence", {length, dropped, pages}, [&](dkv_pool& p) {
    const Sequence* s = p.find(seq, "dkv_pool_sequence");
    if (!s) return DKV_EINVAL;
    *length = s->length, *dropped = s->dropped, *pages = (int32_t)s->pages.size();
    return 0;
  });
}

int64_t dkv_pool_length(dkv_pool* pool, int64_t seq) {
  int64_t length = -1;
  guarded(pool, "dkv_pool_length", {}, [&](dkv_pool& p) {
    const Sequence* s = p.find(seq, "dkv_pool_length");
    if (!s) return DKV_EINVAL;
    length = s->length;
    return 0;
  });
  return length;
}

int dkv_pool_pages(dkv_pool* pool, int64_t seq, int32_t room, uint32_t* page, int32_t* rows, int32_t* holders) {
  return guarded(pool, "dkv_pool_pages", {room > 0 ? (const void*)page : pool, room > 0 ? (const void*)rows : pool, room > 0 ? (const void*)holders : pool}, [&](dkv_pool& p) {
    const Sequence* s = p.find(seq, "dkv_pool_pages");
    if (!s) return DKV_EINVAL;
    if ((size_t)std::max(room, 0) < s->pages.size()) {
      set_error("dkv_pool_pages: room for %d of %zu pages", room, s->pages.size());
      return DKV_EINVAL;
    }
    for (size_t i = 0; i < s->pages.size(); ++i) page[i] = s->pages[i], rows[i] = s->rows[i], holders[i] = p.refs[s->pages[i] >> 2];
    return 0;
  });
}

int dkv_pool_add(dkv_pool* pool, int64_t* seq) {
  return guarded(pool, "dkv_pool_add", {seq}, [&](dkv_pool& p) {
    p.seqs.emplace(p.next, Sequence());
    *seq = p.next++;
    return 0;
  });
}

int dkv_pool_adopt(dkv_pool* pool, const void* src, int64_t src_bytes, const dkv_tile* tiles, int32_t n_tiles, int64_t tokens,
                   int64_t dropped, void* arena, void* stream, int64_t* seq) {
  return guarded(pool, "dkv_pool_adopt", {seq}, [&](dkv_pool& p) {
    const char* what = "dkv_pool_adopt";
    if (n_tiles < 0 || tokens < 0 || dropped < 0 || tokens > INT32_MAX || dropped > INT32_MAX || (n_tiles > 0 && (!tiles || !src))) {
      set_error("%s: bad arguments (tiles %d, tokens %lld, dropped %lld) or a null pointer", what, n_tiles, (long long)tokens, (long long)dropped);
      return DKV_EINVAL;
    }
    // Runs of tiles at one width fill pages one after the other.
    std::vector<dkv_page_move> moves;
    std::vector<int> codes;  // of the pages
    Sequence s;
    int64_t need[3] = {}, at = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const dkv_tile& t = tiles[i];
      const int c = code_of(t.bits), held = (int)std::min<int64_t>(t.rows, tokens - t.token_start);
      if (c < 0 || t.token_start != at || held <= 0 || t.rows > TILE || t.offset < 0 || (t.offset & 15) ||
          t.offset > src_bytes - slab_bytes(t.rows, t.bits, p.layers, p.heads)) {
        set_error("%s: tile %d (%d rows of %d bits at byte %lld, token %d) does not follow the one before it or lies outside its arena", what, i,
                  t.rows, t.bits, (long long)t.offset, t.token_start);
        return DKV_EINVAL;
      }
      at += held;
      for (int r = 0; r < held;) {
        if (codes.empty() || codes.back() != c || s.rows.back() == TILE) codes.push_back(c), s.rows.push_back(0), ++need[c];
        const int n = std::min(held - r, TILE - s.rows.back());
        moves.push_back(dkv_page_move{t.offset, (int64_t)codes.size() - 1, (uint8_t)t.rows, (uint8_t)r, (uint8_t)s.rows.back(), (uint8_t)n,
                                      (uint8_t)t.bits, {}});
        s.rows.back() += n;
        r += n;
      }
    }
    if (at != tokens) {
      set_error("%s: the tiles hold %lld of %lld tokens", what, (long long)at, (long long)tokens);
      return DKV_EINVAL;
    }
    s.pages.reserve(codes.size());
    s.length = tokens, s.dropped = dropped;
    if (int rc = p.make_room(need, arena, stream, what)) return rc;
    auto& mine = p.seqs.emplace(p.next, std::move(s)).first->second;
    for (int c : codes) mine.pages.push_back(p.take(c));
    for (auto& m : moves) m.dst_offset = p.offset(mine.pages[m.dst_offset]);
    if (int rc = launch_moves(src, arena, moves.data(), (int)moves.size(), p.layers, p.heads, stream)) {
      p.release(mine.pages.data(), mine.pages.size());
      p.seqs.erase(p.next);
      return rc;
    }
    *seq = p.next++;
    return 0;
  });
}

int dkv_pool_fork(dkv_pool* pool, int64_t seq, int32_t n, void* arena, void* stream, int64_t* out) {
  return guarded(pool, "dkv_pool_fork", {n > 0 ? (const void*)out : pool}, [&](dkv_pool& p) {
    const char* what = "dkv_pool_fork";
    Sequence* s = p.find(seq, what);
    if (!s) return DKV_EINVAL;
    if (n < 0) {
      set_error("%s: cannot make %d branches", what, n);
      return DKV_EINVAL;
    }
    const bool copies = !s->pages.empty() && s->rows.back() < TILE;  // a last page that is not full is each one's own
    const int c = copies ? s->pages.back() & 3 : 0;
    int64_t need[3] = {};
    if (copies) need[c] = n;
    if (int rc = p.make_room(need, arena, stream, what)) return rc;
    std::vector<dkv_page_move> moves(copies ? n : 0);
    int made = 0;
    auto undo = [&] {
      for (int i = 0; i < made; ++i) {
        const auto it = p.seqs.find(p.next + i);
        p.release(it->second.pages.data(), it->second.pages.size());
        p.seqs.erase(it);
      }
    };
    try {
      for (; made < n; ++made) {
        Sequence copy = *s;
        if (copies) copy.pages.pop_back();
        auto& mine = p.seqs.emplace(p.next + made, std::move(copy)).first->second;
        for (uint32_t page : mine.pages) ++p.refs[page >> 2];
        if (!copies) continue;
        const uint32_t page = p.take(c);
        mine.pages.push_back(page);  // (its room is there: pop_back keeps it)
        moves[made] = dkv_page_move{p.offset(s->pages.back()), p.offset(page), TILE, 0, 0, (uint8_t)s->rows.back(), (uint8_t)(4 << c), {}};
      }
    } catch (...) {
      undo();
      throw;
    }
    if (int rc = launch_moves(arena, arena, moves.data(), (int)moves.size(), p.layers, p.heads, stream)) {
      undo();
      return rc;
    }
    for (int i = 0; i < n; ++i) out[i] = p.next + i;
    p.next += n;
    return 0;
  });
}

int dkv_pool_free(dkv_pool* pool, const int64_t* seqs, int32_t n) {
  return guarded(pool, "dkv_pool_free", {}, [&](dkv_pool& p) {
    std::vector<Sequence*> s;
    if (int rc = p.named(seqs, n, s, "dkv_pool_free")) return rc;
    for (int i = 0; i < n; ++i) {
      p.release(s[i]->pages.data(), s[i]->pages.size());
      p.seqs.erase(seqs[i]);
    }
    if (n) ++p.generation;
    return 0;
  });
}

int dkv_pool_truncate(dkv_pool* pool, int64_t seq, int64_t length, void* arena, void* stream) {
  return guarded(pool, "dkv_pool_truncate", {}, [&](dkv_pool& p) {
    const char* what = "dkv_pool_truncate";
    Sequence* s = p.find(seq, what);
    if (!s) return DKV_EINVAL;
    if (length < 0 || length > s->length) {
      set_error("%s: sequence %lld holds %lld tokens, not %lld", what, (long long)seq, (long long)s->length, (long long)length);
      return DKV_EINVAL;
    }
    if (length == s->length) return 0;
    size_t keep = 0;  // pages that stay
    int64_t held = 0;
    for (; held < length; ++keep) held += s->rows[keep];
    const int last = keep ? (int)(length - (held - s->rows[keep - 1])) : 0;
    if (keep && last < TILE && p.refs[s->pages[keep - 1] >> 2] > 1) {  // others hold it: a sequence appends to a page of its own
      const int c = s->pages[keep - 1] & 3;
      int64_t need[3] = {};
      need[c] = 1;
      // (The copy is made before anything is freed, so that a launch that fails has changed nothing.)
      int64_t first = held;  // the least length whose cut needs no copy
      for (size_t j = keep - 1; s->rows[j] < TILE && p.refs[s->pages[j] >> 2] > 1;) first += s->rows[++j];
      char why[160];
      snprintf(why, sizeof why, first < s->length ? "%s (copies a page that others hold, then frees; cut to %lld first)" : "%s (copies a page that others hold)",
               what, (long long)first);
      if (int rc = p.make_room(need, arena, stream, why)) return rc;
      const uint32_t old = s->pages[keep - 1], page = p.take(c);
      const dkv_page_move move{p.offset(old), p.offset(page), TILE, 0, 0, (uint8_t)last, (uint8_t)(4 << c), {}};
      if (int rc = launch_moves(arena, arena, &move, 1, p.layers, p.heads, stream)) {
        p.release(&page, 1);
        return rc;
      }
      p.release(&old, 1);
      s->pages[keep - 1] = page;
    }
    p.release(s->pages.data() + keep, s->pages.size() - keep);
    s->pages.resize(keep), s->rows.resize(keep);
    if (keep) s->rows.back() = last;
    s->length = length;
    ++p.generation;
    return 0;
  });
}

int dkv_pool_compact(dkv_pool* pool, void* arena, void* stream, int64_t* moved) {
  return guarded(pool, "dkv_pool_compact", {moved}, [&](dkv_pool& p) { return p.compact(arena, stream, *moved); });
}

int64_t dkv_pool_step_bytes(dkv_pool* pool, int32_t n, const int64_t* seqs, const int32_t* counts, const int32_t* bits, int64_t reserve,
                            int32_t* max_pages) {
  int64_t bytes = 0;
  const int rc = guarded(pool, "dkv_pool_step_bytes", {max_pages}, [&](dkv_pool& p) {
    Ask a;
    if (int rc = read_ask(p, n, seqs, counts, bits, a, "dkv_pool_step_bytes")) return rc;
    // a page that is begun and those that the reserve fills, of every sequence
    const int64_t most = a.pages + (reserve > 0 ? n * ((reserve + TILE - 1) / TILE + 1) : 0);
    if (reserve < 0 || most > INT32_MAX / 4) {
      set_error("dkv_pool_step_bytes: a reserve of %lld tokens", (long long)reserve);
      return DKV_EINVAL;
    }
    const std::vector<int32_t> zero(n + 1, 0);
    const dkv_paged_batch b{n, counts, zero.data(), zero.data(), zero.data(), nullptr, nullptr, p.layers, p.heads, p.q_heads, 0, (int32_t)most,
                            p.precision};
    bytes = dkv_paged_plan_bytes(&b);
    *max_pages = (int32_t)most;
    return bytes ? 0 : DKV_EINVAL;
  });
  return rc ? 0 : bytes;
}

int dkv_pool_step(dkv_pool* pool, int32_t n, const int64_t* seqs, const int32_t* counts, const int32_t* bits, int32_t max_pages, void* arena,
                  void* stream, void* buffer, int64_t bytes, dkv_paged_plan* plan, int64_t* generation) {
  return guarded(pool, "dkv_pool_step", {plan, generation}, [&](dkv_pool& p) {
    const char* what = "dkv_pool_step";
    Ask a;
    if (int rc = read_ask(p, n, seqs, counts, bits, a, what)) return rc;
    if (a.pages > max_pages) {
      set_error("%s: the sequences have %lld pages, the plan has room for %d", what, (long long)a.pages, max_pages);
      return DKV_EINVAL;
    }
    if (int rc = p.make_room(a.need, arena, stream, what)) return rc;
    std::vector<int32_t> past(n), position(n), first(n + 1, 0), rows;
    std::vector<uint32_t> pages;
    std::vector<std::pair<size_t, int>> old(n);  // pages, and rows of the last one, before
    pages.reserve(a.pages), rows.reserve(a.pages);
    for (int i = 0; i < n; ++i) {
      Sequence& s = *a.s[i];
      s.pages.reserve(s.pages.size() + s.fresh(counts[i], a.code[i])), s.rows.reserve(s.pages.capacity());
      old[i] = {s.pages.size(), s.rows.empty() ? 0 : s.rows.back()};
      past[i] = (int32_t)s.length, position[i] = (int32_t)(s.length + s.dropped);
    }
    int grown = 0;
    auto undo = [&] {
      for (int i = 0; i < grown; ++i) {
        Sequence& s = *a.s[i];
        p.release(s.pages.data() + old[i].first, s.pages.size() - old[i].first);
        s.pages.resize(old[i].first), s.rows.resize(old[i].first);
        if (old[i].first) s.rows.back() = old[i].second;
        s.length = past[i];
      }
    };
    int rc;
    try {
      for (; grown < n; ++grown) {
        Sequence& s = *a.s[grown];
        int left = counts[grown];
        const int here = std::min(s.room(a.code[grown]), left);
        if (here > 0) s.rows.back() += here, left -= here;
        for (; left > 0; left -= TILE) s.pages.push_back(p.take(a.code[grown])), s.rows.push_back(std::min(left, TILE));
        s.length += counts[grown];
        pages.insert(pages.end(), s.pages.begin(), s.pages.end());
        rows.insert(rows.end(), s.rows.begin(), s.rows.end());
        first[grown + 1] = (int32_t)pages.size();
      }
      const dkv_paged_batch b{n, counts, past.data(), position.data(), first.data(), pages.data(), rows.data(), p.layers, p.heads, p.q_heads,
                              p.blocks * BLOCK * p.grain, max_pages, p.precision};
      rc = dkv_paged_plan_write(&b, buffer, bytes, plan);
    } catch (...) {
      grown = std::min(grown + 1, n);  // (the one that was growing among them)
      undo();
      throw;
    }
    if (rc) undo();
    *generation = p.generation;
    return rc;
  });
}

int64_t dkv_pool_tokens(dkv_pool* pool, int32_t n, const int64_t* seqs, const int64_t* from) {
  int64_t total = 0;
  const int rc = guarded(pool, "dkv_pool_tokens", {n > 0 ? (const void*)from : pool}, [&](dkv_pool& p) {
    std::vector<Sequence*> s;
    if (int rc = p.named(seqs, n, s, "dkv_pool_tokens")) return rc;
    for (int i = 0; i < n; ++i) {
      if (from[i] < 0 || from[i] > s[i]->length) {
        set_error("dkv_pool_tokens: sequence %lld holds %lld tokens, not %lld", (long long)seqs[i], (long long)s[i]->length, (long long)from[i]);
        return DKV_EINVAL;
      }
      total += s[i]->length - from[i];
    }
    if (total > INT32_MAX) {
      set_error("dkv_pool_tokens: %lld tokens are too many for one tensor", (long long)total);
      return DKV_EINVAL;
    }
    return 0;
  });
  return rc ? -1 : total;
}

int dkv_pool_read(dkv_pool* pool, int32_t n, const int64_t* seqs, const int64_t* from, int32_t layer0, int32_t n_layers, const void* arena,
                  void* out, int32_t n_tokens, int32_t out_dtype, void* stream) {
  // (Launched under the lock: a call that moves or frees the pages is enqueued before they are looked up or behind the reads.)
  return guarded(pool, "dkv_pool_read", {n > 0 ? (const void*)from : pool}, [&](dkv_pool& p) {
    const char* what = "dkv_pool_read";
    std::vector<dkv_page_rows> items;
    std::vector<Sequence*> s;
    if (int rc = p.named(seqs, n, s, what)) return rc;
    int64_t to = 0;
    for (int i = 0; i < n; ++i) {
      if (from[i] < 0 || from[i] > s[i]->length) {
        set_error("%s: sequence %lld holds %lld tokens, not %lld", what, (long long)seqs[i], (long long)s[i]->length, (long long)from[i]);
        return DKV_EINVAL;
      }
      int64_t at = 0;
      for (size_t j = 0; j < s[i]->pages.size(); at += s[i]->rows[j++]) {
        const int row0 = (int)std::min<int64_t>(std::max<int64_t>(from[i] - at, 0), s[i]->rows[j]), rows = s[i]->rows[j] - row0;
        if (rows > 0) items.push_back(dkv_page_rows{(int32_t)to, s[i]->pages[j], row0, rows}), to += rows;
      }
    }
    if (to != n_tokens) {
      set_error("%s: room for %d tokens, not %lld", what, n_tokens, (long long)to);
      return DKV_EINVAL;
    }
    return dkv_paged_read(arena, p.blocks * BLOCK * p.grain, items.data(), (int32_t)items.size(), layer0, n_layers, p.layers, p.heads, out,
                          n_tokens, out_dtype, stream);
  });
}

}  // extern "C"
