"""Packed mixed-precision KV cache of many sequences, in pages that sequences share.

A GPUCache holds one sequence, and its forks run one after another. A PagedCache holds any number of them in one HBM
arena: a sequence is a list of pages of 64 tokens at 4, 8 or 16 bits, branches share the pages that they have in
common, and one launch packs or attends for all sequences of a step, whatever their lengths. The packed rows are
GPUCache's, byte for byte (include/dkv.h). No counterpart in the reference, whose cache holds one sequence.

    cache = PagedCache(layers, heads, q_heads, max_tokens=1 << 20)
    stream = cache.adopt(gpu_cache)             # an ingested GPUCache's history, as it is packed
    seqs = cache.fork(stream, 4)                # four questions about it
    step = cache.step(seqs, [12, 7, 31, 9])     # their tokens, one sequence after the other
    for layer in range(layers):                 # q [1, q_heads, 59, 64], k and v [1, heads, 59, 64]
        cache.append(k, v, layer, step)
        out = cache.attend(q, k, v, layer, step)  # [1, 59, q_heads, 64]
    step = cache.step(seqs)                     # the next token of each
"""
import ctypes
import heapq
import struct

import numpy as np
import torch

from . import _lib
from .gpu_cache import BITS, OUT_DTYPES, PRECISIONS, TILE, GPUCache, _check_dtype

try:  # transformers passes a cache that is one of its own through its decoder
    from transformers.cache_utils import DynamicCache as _CacheBase
except Exception:
    _CacheBase = object

GRAINS = {4: 5, 8: 9, 16: 16}  # grains (dkv_page_grain) of a page
CODE = {4: 0, 8: 1, 16: 2}
# The arena is cut into blocks of 48 grains that hold pages of one width while they hold any: 9, 5 or 3 of them, of
# which 45, 45 or 48 grains are used. So no free room is too small for any page but within a block, and the pages of a
# width can be brought together into as few blocks as hold them (compact()).
BLOCK = 48
PER_BLOCK = {w: BLOCK // g for w, g in GRAINS.items()}
FULL = {w: (1 << n) - 1 for w, n in PER_BLOCK.items()}
MOVE_DTYPE = np.dtype([('src', '<i8'), ('dst', '<i8'), ('src_rows', 'u1'), ('src_row', 'u1'), ('dst_row', 'u1'),
                       ('rows', 'u1'), ('bits', 'u1'), ('reserved', 'u1', 3)])
ROWS_DTYPE = np.dtype([('token', '<i4'), ('page', '<u4'), ('row0', '<i4'), ('rows', '<i4')])
_PLAN_BYTES = ctypes.sizeof(_lib.PagedPlan)
_ARGS = struct.Struct(f'PqqPqqPqqPqP{_PLAN_BYTES}siifPqqiiPq')  # dkv_paged_args, with the plan as bytes
assert _ARGS.size == ctypes.sizeof(_lib.PagedArgs) and MOVE_DTYPE.itemsize == 24 and ROWS_DTYPE.itemsize == 16
_NONE = np.zeros(0, dtype=np.uint32)


def _width(page):
    return 4 << (page & 3)


class _Sequence:
    __slots__ = ('pages', 'rows', 'length', 'dropped')

    def __init__(self, pages=_NONE, rows=None, length=0, dropped=0):
        self.pages = pages  # dkv_page words in token order; replaced, never written
        self.rows = np.zeros(0, dtype=np.int32) if rows is None else rows  # tokens of each
        self.length, self.dropped = length, dropped

    def room(self, bits):
        """Rows that the last page has left for tokens of this width."""
        n = len(self.pages)
        return TILE - int(self.rows[n - 1]) if n and _width(int(self.pages[n - 1])) == bits else 0

    def grow(self, n, bits, fresh):
        """n more tokens: what the last page has room for, the rest in `fresh` pages. Returns how many the last took."""
        first = min(self.room(bits), n)
        rows = np.concatenate((self.rows, np.full(len(fresh), TILE, dtype=np.int32)))
        if first:
            rows[len(self.rows) - 1] += first
        if fresh:
            rows[-1] = n - first - TILE * (len(fresh) - 1)
            self.pages = np.concatenate((self.pages, np.array(fresh, dtype=np.uint32)))
        self.rows, self.length = rows, self.length + n
        return first


class PagedCache:
    """Mixed 4/8/16-bit KV cache of many sequences, head_dim 64. Sequences are named by the ints that add(), adopt()
    and fork() return.

    max_tokens: room for that many tokens at 16 bits in full pages (some more at 8, three times as many at 4); a
    sequence's last page, and one after which the width changes, may be part full. precision as in GPUCache.
    The calls on one cache belong on one stream, or on streams that wait for each other: pages that a call frees are
    written again by later ones.
    """

    def __init__(self, layers, heads, q_heads, max_tokens=8192, dim=64, device='cuda', precision='bf16', arena_bytes=None):
        if dim != 64:
            raise ValueError('GPU kernel currently supports head_dim=64')
        if precision not in PRECISIONS:
            raise ValueError(f'precision must be one of {sorted(PRECISIONS)}')
        if layers < 1 or heads < 1 or q_heads < 1 or q_heads % heads:
            raise ValueError(f'PagedCache: q_heads must be a multiple of heads, got {layers} layers, {heads} of {q_heads} heads')
        self.layers, self.heads, self.q_heads, self.dim, self.precision = layers, heads, q_heads, dim, precision
        self.device = torch.device(device)
        self.grain = 512 * 2 * layers * heads
        block = BLOCK * self.grain
        if arena_bytes is None:
            arena_bytes = -(-max(max_tokens, 1) // (TILE * PER_BLOCK[16])) * block
        self.blocks = int(arena_bytes) // block
        if not 1 <= self.blocks <= (1 << 30) // BLOCK - 1:
            raise ValueError(f'PagedCache: an arena of {arena_bytes} bytes holds {self.blocks} blocks of {block}')
        self.arena_bytes = self.blocks * block
        with torch.inference_mode(False):
            self.arena = torch.empty(self.arena_bytes, dtype=torch.uint8, device=self.device)
        self._width = [0] * self.blocks  # of a block's pages; 0: it holds none
        self._used = [0] * self.blocks  # bits of the pages that it holds
        self._empty = list(range(self.blocks))  # heap of blocks without pages
        self._partial = {w: [] for w in BITS}  # heaps of blocks with room (and some that had it)
        self._n_blocks = {w: 0 for w in BITS}
        self._n_pages = {w: 0 for w in BITS}
        self._refs = np.zeros(self.blocks * BLOCK, dtype=np.int32)  # sequences that hold the page at a grain
        self._seqs = {}
        self._next = 0
        self._generation = 0  # of steps: pages were freed, cut or moved since

    # -- pages -----------------------------------------------------------------
    def _take(self, bits):
        heap = self._partial[bits]
        while heap and not (self._width[heap[0]] == bits and self._used[heap[0]] != FULL[bits]):
            heapq.heappop(heap)
        if heap:
            block = heap[0]
        else:
            block = heapq.heappop(self._empty)
            self._width[block] = bits
            self._n_blocks[bits] += 1
            heapq.heappush(heap, block)
        free = ~self._used[block] & FULL[bits]
        slot = (free & -free).bit_length() - 1
        self._used[block] |= 1 << slot
        self._n_pages[bits] += 1
        grain = block * BLOCK + slot * GRAINS[bits]
        self._refs[grain] = 1
        return grain << 2 | CODE[bits]

    def _give(self, page):
        bits, grain = _width(page), page >> 2
        block = grain // BLOCK
        if self._used[block] == FULL[bits]:
            heapq.heappush(self._partial[bits], block)
        self._used[block] &= ~(1 << (grain % BLOCK) // GRAINS[bits])
        self._n_pages[bits] -= 1
        if not self._used[block]:
            self._width[block] = 0
            self._n_blocks[bits] -= 1
            heapq.heappush(self._empty, block)

    def _release(self, pages):
        """One holder less of each page; those without one go back."""
        at = pages >> 2
        self._refs[at] -= 1
        for page in pages[self._refs[at] == 0].tolist():
            self._give(page)

    def _make_room(self, need):
        """Room for need[w] new pages of each width: pages are brought together if that makes it."""
        def blocks(extra):  # that hold what there is and what is needed
            return sum(max(-(-(self._n_pages[w] + need.get(w, 0)) // PER_BLOCK[w]), self._n_blocks[w] * extra) for w in BITS)
        if blocks(1) <= self.blocks:
            return
        if blocks(0) > self.blocks:
            have = {w: self._n_pages[w] for w in BITS}
            raise ValueError(f'paged cache is full: {need} new pages by width beside {have} in {self.blocks} blocks')
        self.compact()

    def _call(self, name, *args):
        """One C entry point on this cache's device and torch's current stream there."""
        if not self.arena.is_cuda:
            raise ValueError('PagedCache requires a CUDA device')
        index = self.arena.get_device()
        fn = getattr(_lib.load(), name)
        if torch.cuda.current_device() == index:
            rc = fn(*args, _lib.raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, _lib.raw_stream(index))
        if rc:
            _lib.check(rc, name)

    def _move(self, source, moves):
        if moves:
            moves = np.array(moves, dtype=MOVE_DTYPE)
            self._call('dkv_paged_move', source.data_ptr(), source.numel(), self.arena.data_ptr(), self.arena_bytes,
                       moves.ctypes.data, len(moves), self.layers, self.heads)

    def _page_move(self, page, to, rows):
        """A whole page's first rows to another page of its width."""
        return ((page >> 2) * self.grain, (to >> 2) * self.grain, TILE, 0, 0, rows, _width(page), (0, 0, 0))

    def _not_captured(self, what):
        if self.arena.is_cuda and torch.cuda.is_current_stream_capturing():
            raise ValueError(f'{what} cannot run while a graph is captured')

    # -- sequences -------------------------------------------------------------
    def _sequence(self, seq):
        try:
            return self._seqs[seq]
        except (KeyError, TypeError):
            raise ValueError(f'no sequence {seq!r} in this cache') from None

    def _named(self, seqs, what):
        """A list of distinct sequences of this cache from one or several."""
        seqs = [seqs] if isinstance(seqs, (int, np.integer)) else list(seqs)
        for seq in seqs:
            self._sequence(seq)
        if len(set(seqs)) != len(seqs):
            raise ValueError(f'{what}: a sequence is named twice')
        return seqs

    def _new(self, sequence):
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = sequence
        return seq

    def add(self):
        """A new, empty sequence."""
        return self._new(_Sequence())

    def length(self, seq):
        """Tokens that a sequence holds, those of steps that were planned among them."""
        return self._sequence(seq).length

    def position(self, seq):
        """Position of a sequence's next token: its length and what an evicted GPUCache that it was adopted from had
        dropped."""
        s = self._sequence(seq)
        return s.length + s.dropped

    def adopt(self, cache):
        """A new sequence with the history of a GPUCache (all layers level): its packed rows are copied as they are,
        gathered into pages."""
        if not isinstance(cache, GPUCache):
            raise ValueError('adopt expects a GPUCache')
        if cache.layers != self.layers or cache.heads != self.heads or cache.arena.device != self.arena.device:
            raise ValueError(f'adopt: {cache.layers} layers of {cache.heads} heads on {cache.arena.device} do not go into '
                             f'{self.layers} of {self.heads} on {self.arena.device}')
        if len(set(cache.seen)) != 1:
            raise ValueError('adopt: every layer must be at the same length')
        self._not_captured('adopt')
        n = cache.seen[0]
        tiles = cache.tiles_host[:cache._tiles_before(n)]
        # runs of tiles at one width fill pages one after the other
        offsets, starts, widths = tiles['offset'].tolist(), tiles['token_start'].tolist(), tiles['bits'].tolist()
        layout = tiles['rows'].tolist()
        held = [min(r, n - t) for r, t in zip(layout, starts)]
        room, need, bits = 0, {w: 0 for w in BITS}, 0
        for w, r in zip(widths, held):
            room = room if w == bits else 0
            fresh = -(-(r - room) // TILE) if r > room else 0
            need[w] += fresh
            room, bits = room + fresh * TILE - r, w
        self._make_room(need)
        moves, pages, rows, bits = [], [], [], 0
        for offset, w, size, r in zip(offsets, widths, layout, held):
            at = 0
            while at < r:
                if w != bits or rows[-1] == TILE:
                    pages.append(self._take(w))
                    rows.append(0)
                    bits = w
                m = min(r - at, TILE - rows[-1])
                moves.append((offset, (pages[-1] >> 2) * self.grain, size, at, rows[-1], m, w, (0, 0, 0)))
                rows[-1] += m
                at += m
        self._move(cache.arena, moves)
        return self._new(_Sequence(np.array(pages, dtype=np.uint32), np.array(rows, dtype=np.int32), n, cache.dropped))

    def fork(self, seq, n=1):
        """n new sequences that go on from this one. They share its pages but a last one that is not full, of which
        each gets a copy."""
        s = self._sequence(seq)
        if n < 0:
            raise ValueError(f'fork: cannot make {n} branches')
        self._not_captured('fork')
        part = len(s.pages) > 0 and s.rows[-1] < TILE
        if part:
            self._make_room({_width(int(s.pages[-1])): n})
        whole = s.pages[:-1] if part else s.pages
        self._refs[whole >> 2] += n
        out, moves = [], []
        for _ in range(n):
            pages = s.pages
            if part:
                last = int(pages[-1])
                copy = self._take(_width(last))
                moves.append(self._page_move(last, copy, int(s.rows[-1])))
                pages = np.concatenate((whole, np.array([copy], dtype=np.uint32)))
            out.append(self._new(_Sequence(pages, s.rows.copy(), s.length, s.dropped)))
        self._move(self.arena, moves)
        return out

    def free(self, seqs):
        """Ends sequences; pages that no other one holds are free again."""
        self._not_captured('free')
        for seq in self._named(seqs, 'free'):
            self._release(self._seqs.pop(seq).pages)
            self._generation += 1

    def truncate(self, seq, length):
        """Drops a sequence's tokens from `length` on."""
        s = self._sequence(seq)
        if not 0 <= length <= s.length:
            raise ValueError(f'truncate: sequence {seq} holds {s.length} tokens, not {length}')
        if length == s.length:
            return
        self._not_captured('truncate')
        ends = np.cumsum(s.rows)
        keep = int(np.searchsorted(ends, length))  # pages before the one that holds the last token that stays
        rows = s.rows[:keep + 1].copy() if length else s.rows[:0]
        pages, gone = s.pages[:len(rows)], s.pages[len(rows):]
        if length:
            rows[-1] = length - (int(ends[keep - 1]) if keep else 0)
            if rows[-1] < TILE and self._refs[pages[-1] >> 2] > 1:  # others hold it: a sequence appends to a page of its own
                self._make_room({_width(int(pages[-1])): 1})
                pages, gone = s.pages[:len(rows)], s.pages[len(rows):]  # (moved, if pages were brought together)
                copy = self._take(_width(int(pages[-1])))
                self._move(self.arena, [self._page_move(int(pages[-1]), copy, int(rows[-1]))])
                gone = s.pages[len(rows) - 1:]
                pages = np.concatenate((pages[:-1], np.array([copy], dtype=np.uint32)))
        s.pages, s.rows, s.length = pages, rows, length
        self._release(gone)
        self._generation += 1

    def compact(self):
        """Brings the pages of each width together into as few blocks as hold them: what was free in pieces can hold
        pages of any width. Returns how many pages were moved. (Calls that find too little room do it themselves.)
        Steps that were planned before have to be planned again."""
        self._not_captured('compact')
        moves, old, new = [], [], []
        for w in BITS:
            held = sorted((b for b in range(self.blocks) if self._width[b] == w), key=lambda b: (-self._used[b].bit_count(), b))
            target = -(-self._n_pages[w] // PER_BLOCK[w])
            free = [(b, s) for b in held[:target] for s in range(PER_BLOCK[w]) if not self._used[b] >> s & 1]
            at = 0
            for b in held[target:]:
                for s in range(PER_BLOCK[w]):
                    if self._used[b] >> s & 1:
                        (to, slot), at = free[at], at + 1
                        old.append(b * BLOCK + s * GRAINS[w])
                        new.append(to * BLOCK + slot * GRAINS[w])
                        moves.append((old[-1] * self.grain, new[-1] * self.grain, TILE, 0, 0, TILE, w, (0, 0, 0)))
                        self._used[to] |= 1 << slot
                self._used[b], self._width[b] = 0, 0
                self._n_blocks[w] -= 1
                heapq.heappush(self._empty, b)
            self._partial[w] = [b for b in held[:target] if self._used[b] != FULL[w]]
            heapq.heapify(self._partial[w])
        if not moves:
            return 0
        self._move(self.arena, moves)
        old, new = np.array(old), np.array(new)
        self._refs[new] = self._refs[old]
        self._refs[old] = 0
        to = np.arange(len(self._refs), dtype=np.uint32)
        to[old] = new
        for s in self._seqs.values():
            s.pages = to[s.pages >> 2] << 2 | s.pages & 3
        self._generation += 1
        return len(moves)

    def accounting(self):
        """Pages by width, and bytes: of the arena, of blocks that hold pages, and of the pages."""
        return dict(sequences=len(self._seqs), pages=dict(self._n_pages), allocated_bytes=self.arena_bytes,
                    block_bytes=sum(self._n_blocks.values()) * BLOCK * self.grain,
                    page_bytes=sum(GRAINS[w] * n for w, n in self._n_pages.items()) * self.grain,
                    free_blocks=len(self._empty))

    # -- steps -----------------------------------------------------------------
    def step(self, seqs, counts=1, bits=16, reserve=0):
        """The next tokens of some sequences: `counts` of each (one number or one a sequence), at width `bits` (too).
        Opens their pages and plans what every layer's append() and attend() do; the sequences are as long from here
        on. The step's tensors hold the sequences' tokens one after the other, in this order. `reserve`: room in the
        plan for as many more tokens of every sequence, for steps that go on with advance(). Sequences that share
        pages attend to these together where they stand next to each other."""
        return PagedStep(self, seqs, counts, bits, reserve)

    def _grow(self, seqs, counts, bits):
        """Room for the tokens of a step, all or none."""
        need = {w: 0 for w in BITS}
        for seq, n, w in zip(seqs, counts, bits):
            need[w] += max(-(-(n - self._seqs[seq].room(w)) // TILE), 0)
        self._make_room(need)
        for seq, n, w in zip(seqs, counts, bits):
            s = self._seqs[seq]
            s.grow(n, w, [self._take(w) for _ in range(max(-(-(n - s.room(w)) // TILE), 0))])

    def _check(self, what, step, layer, tensors):
        if not isinstance(step, PagedStep) or step.cache is not self:
            raise ValueError(f'{what} expects a step of this cache')
        if step.generation != self._generation:
            raise ValueError(f'{what}: pages were freed, cut or moved since this step was planned')
        if not 0 <= layer < self.layers:
            raise ValueError(f'{what}: layer {layer} of {self.layers}')
        index = self.arena.get_device()
        for x, heads in tensors:
            if x.dim() != 4 or x.shape != (1, heads, step.tokens, self.dim):
                raise ValueError(f'{what} expects [1, {heads}, {step.tokens}, {self.dim}], got {list(x.shape)}')
            if index < 0 or x.get_device() != index:
                raise ValueError(f'{what} requires CUDA tensors on the device of the cache')

    def append(self, k, v, layer, step):
        """Packs the step's new tokens of one layer, k and v [1, heads, tokens, 64], into their pages."""
        self._check('append', step, layer, ((k, self.heads), (v, self.heads)))
        k, kp, ks = GPUCache._rows(k)
        v, vp, vs = GPUCache._rows(v)
        self._call('dkv_paged_append', _ARGS.pack(0, 0, 0, kp, ks[1], ks[2], vp, vs[1], vs[2], self.arena.data_ptr(), self.arena_bytes,
                                                  step.device_plan(), step.plan_bytes, layer, step.captured(), 0.0, 0, 0, 0, 0, 0, 0, 0))

    def attend(self, q, k, v, layer, step, out_dtype=None, precision=None):
        """Causal attention of the step's tokens, q [1, q_heads, tokens, 64], each over its sequence's history and the
        sequence's new tokens k, v [1, heads, tokens, 64] up to itself (these as they are, not as they are packed;
        append() may come before or after). Returns [1, tokens, q_heads, 64] in out_dtype (default q's)."""
        precision = precision or self.precision
        if precision not in PRECISIONS:
            raise ValueError(f'precision must be one of {sorted(PRECISIONS)}')
        out_dtype = out_dtype or q.dtype
        if out_dtype not in OUT_DTYPES:
            _check_dtype(out_dtype, 'attend output dtype')
        self._check('attend', step, layer, ((q, self.q_heads), (k, self.heads), (v, self.heads)))
        q, qp, qs = GPUCache._rows(q)
        k, kp, ks = GPUCache._rows(k)
        v, vp, vs = GPUCache._rows(v)
        out = q.new_empty((1, step.tokens, self.q_heads, self.dim), dtype=out_dtype)
        bounds = step.captured()
        need = step.workspace_bytes(bounds)
        ws = self.arena.new_empty(need) if need else None
        self._call('dkv_paged_attend', _ARGS.pack(
            qp, qs[1], qs[2], kp, ks[1], ks[2], vp, vs[1], vs[2], self.arena.data_ptr(), self.arena_bytes, step.device_plan(),
            step.plan_bytes, layer, bounds, self.dim ** -0.5, out.data_ptr(), self.q_heads * self.dim, self.dim,
            out_dtype is torch.float32, PRECISIONS[precision], ws.data_ptr() if need else 0, need))
        return out

    def materialize(self, layer, seqs, first=0, out_dtype=torch.bfloat16):
        """Dequantized tokens of one layer (None: of all), one sequence after the other: (k, v), each [1, heads,
        tokens, 64] ([layers, heads, tokens, 64]). `seqs`: sequences, of which the tokens from `first` on (one number
        or one a sequence), or a step, whose new tokens they are."""
        _check_dtype(out_dtype, 'materialize output dtype')
        if layer is not None and not 0 <= layer < self.layers:
            raise ValueError(f'materialize: layer {layer} of {self.layers}')
        self._not_captured('materialize')  # (a replay would read the pages of now)
        if isinstance(seqs, PagedStep):
            self._check('materialize', seqs, 0, ())
            items, n = seqs.items, seqs.tokens
        else:
            items, n = self._items(self._named(seqs, 'materialize'), first)
        layers = self.layers if layer is None else 1
        out = self.arena.new_empty((2, layers, self.heads, n, self.dim), dtype=out_dtype)
        if n:
            self._call('dkv_paged_read', self.arena.data_ptr(), self.arena_bytes, items.ctypes.data, len(items), layer or 0, layers,
                       self.layers, self.heads, out.data_ptr(), n, int(out_dtype is torch.float32))
        return out[0], out[1]

    def _items(self, seqs, first):
        """(records, tokens) of the sequences' tokens from `first` on."""
        firsts = [first] * len(seqs) if isinstance(first, (int, np.integer)) else list(first)
        if len(firsts) != len(seqs):
            raise ValueError('materialize: one first token a sequence')
        parts, n = [], 0
        for seq, at in zip(seqs, firsts):
            s = self._seqs[seq]
            if not 0 <= at <= s.length:
                raise ValueError(f'materialize: sequence {seq} holds {s.length} tokens, not {at}')
            ends = np.cumsum(s.rows)
            skip = int(np.searchsorted(ends, at, side='right'))
            rows = np.zeros(len(ends) - skip, dtype=ROWS_DTYPE)
            start = ends[skip:] - s.rows[skip:]
            rows['row0'] = np.maximum(at - start, 0)
            rows['rows'] = s.rows[skip:] - rows['row0']
            rows['page'] = s.pages[skip:]
            rows['token'] = n + start + rows['row0'] - at
            n += s.length - at
            parts.append(rows)
        return np.concatenate(parts) if parts else np.zeros(0, dtype=ROWS_DTYPE), n


class PagedStep(_CacheBase):
    """The new tokens of some sequences of a PagedCache (PagedCache.step()), and what the launches over them read.

    positions: [tokens] int64 on the device, of every new token. A step can be the `past_key_values` of a decoder that
    install_packed_attention() patched: its attention then packs and attends for all the sequences. A step that a graph
    capture records can go on: advance() plans the sequences' next tokens into the same device memory, and a replay of
    the graph runs over them.
    """

    backend = 'fused'
    fast_gqa = False

    def __init__(self, cache, seqs, counts, bits, reserve):
        if _CacheBase is not object:
            super().__init__()
        self.cache, self.heads, self.layers = cache, cache.heads, cache.layers
        self.seqs = cache._named(seqs, 'step')

        def each(x, what):
            x = [x] * len(self.seqs) if isinstance(x, (int, np.integer)) else list(x)
            if len(x) != len(self.seqs):
                raise ValueError(f'step: one {what} a sequence')
            return [int(v) for v in x]
        self.counts, self.bits = each(counts, 'count'), each(bits, 'width')
        if not self.seqs or min(self.counts) < 1:
            raise ValueError('step expects sequences and at least one new token of each')
        if set(self.bits) - set(BITS):
            raise ValueError(f'step: widths must be of {BITS}, got {self.bits}')
        if reserve < 0:
            raise ValueError(f'step: reserve must not be negative, got {reserve}')
        if not cache.arena.is_cuda:
            raise ValueError('PagedCache requires a CUDA device')
        cache._not_captured('step')
        self.tokens = sum(self.counts)
        self.reserve = reserve
        self._dev = None
        self._plan(first=True)

    def _plan(self, first=False):
        cache = self.cache
        kept = [(s, s.pages, s.rows, s.length) for s in map(cache._seqs.get, self.seqs)]
        self.past = [s.length for s, _, _, _ in kept]
        position = [s.length + s.dropped for s, _, _, _ in kept]
        cache._grow(self.seqs, self.counts, self.bits)
        try:
            self._write([s for s, _, _, _ in kept], position, first)
        except ValueError:
            for (s, pages, rows, length) in kept:  # as they were
                cache._release(s.pages[len(pages):])
                s.pages, s.rows, s.length = s.pages[:len(pages)], rows, length
            raise
        self.generation = cache._generation

    def _write(self, seqs, position, first):
        cache, lib = self.cache, _lib.load()
        n_pages = [len(s.pages) for s in seqs]
        bounds = np.zeros(len(seqs) + 1, dtype=np.int32)
        np.cumsum(n_pages, out=bounds[1:])
        if first:
            self.max_pages = int(bounds[-1]) + (len(seqs) * (-(-self.reserve // TILE) + 1) if self.reserve else 0)
        pages, rows = np.concatenate([s.pages for s in seqs]), np.concatenate([s.rows for s in seqs])
        ints = np.array([self.counts, self.past, position], dtype=np.int32)
        batch = _lib.PagedBatch(len(seqs), ints[0].ctypes.data, ints[1].ctypes.data, ints[2].ctypes.data, bounds.ctypes.data,
                                pages.ctypes.data, rows.ctypes.data, cache.layers, cache.heads, cache.q_heads, cache.arena_bytes,
                                self.max_pages)
        need = lib.dkv_paged_plan_bytes(ctypes.byref(batch))
        with torch.inference_mode(False):
            # (pinned memory goes back to torch's cache when the copy that reads it is done)
            host = torch.empty(max(need, 16), dtype=torch.uint8, pin_memory=True)
            plan = _lib.PagedPlan()
            _lib.check(lib.dkv_paged_plan_write(ctypes.byref(batch), host.data_ptr(), need, ctypes.byref(plan)), 'dkv_paged_plan_write')
            if self._dev is None:
                self._dev = torch.empty(need, dtype=torch.uint8, device=cache.device)
                self._stream = _lib.raw_stream(cache.device)
            self._dev.copy_(host, non_blocking=True)
        self.plan, self.plan_bytes = plan, bytes(plan)
        at = 4 * plan.at_items
        self.items = host.numpy()[at:at + 16 * plan.items].view(ROWS_DTYPE).copy()
        at = 4 * plan.at_positions
        self.positions = self._dev[at:at + 8 * self.tokens].view(torch.int64)
        self._needs = {}

    def advance(self):
        """Plans the same sequences' next tokens, as many of each and at the same widths, in place of this step's. The
        launches that a capture recorded over this step run over them when they are replayed. The pages that this
        takes must fit into the room of the plan (step(..., reserve=))."""
        for seq in self.seqs:
            self.cache._sequence(seq)
        self.cache._not_captured('advance')
        past, plan = self.past, (self.plan, self.plan_bytes, self.items)
        try:
            self._plan()
        except ValueError:
            self.past = past
            self.plan, self.plan_bytes, self.items = plan
            raise
        return self

    def device_plan(self):
        stream = _lib.raw_stream(self.cache.device)
        if stream != self._stream:  # (its memory is not given out again before that stream is done with it)
            self._dev.record_stream(torch.cuda.current_stream(self.cache.device))
        return self._dev.data_ptr()

    def captured(self):
        """Whether launches are being recorded, which then are sized for every plan that advance() may write."""
        return int(torch.cuda.is_current_stream_capturing())

    def workspace_bytes(self, bounds):
        need = self._needs.get(bounds)
        if need is None:
            args = _lib.PagedArgs(plan=self.plan, bounds=bounds)
            need = self._needs[bounds] = _lib.load().dkv_paged_workspace_bytes(ctypes.byref(args))
        return need

    # -- as the cache of a patched decoder (install_packed_attention) ------------
    def append_projection(self, qkv, cos, sin, q_heads, layer):
        return None  # (no launch of its own: split and RoPE, then append())

    def append(self, k, v, layer):
        self.cache.append(k, v, layer, self)
        return 0

    def attend(self, q, k, v, layer, past=0, **kw):
        return self.cache.attend(q, k, v, layer, self, **kw)

    def get_seq_length(self, layer_idx=0):
        return 0

    def get_max_cache_shape(self, layer_idx=0):
        return None

    def __len__(self):
        return self.layers

    @property
    def is_sliding(self):
        return [False] * self.layers

    @property
    def is_compileable(self):
        return False

    def get_query_offset(self, layer_idx=0):
        return 0

    def get_mask_sizes(self, query_length, layer_idx=0):
        if isinstance(query_length, torch.Tensor):
            query_length = query_length.shape[0]
        return query_length, 0
