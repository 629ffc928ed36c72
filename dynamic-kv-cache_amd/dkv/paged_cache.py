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
import operator
import struct
import threading
import weakref

import numpy as np
import torch

from . import _lib
from .gpu_cache import OUT_DTYPES, PRECISIONS, TILE, GPUCache, _check_dtype

try:  # transformers passes a cache that is one of its own through its decoder
    from transformers.cache_utils import DynamicCache as _CacheBase
except Exception:
    _CacheBase = object

BLOCK, BLOCK_TOKENS = 48, 3 * TILE  # grains of a block of pages; tokens that it holds at 16 bits
IDS = 1 << 62  # sequences' names are below
_PLAN_BYTES = ctypes.sizeof(_lib.PagedPlan)
_ARGS = struct.Struct(f'PqqPqqPqqPqP{_PLAN_BYTES}siifPqqiiPq')  # dkv_paged_args, with the plan as bytes
assert _ARGS.size == ctypes.sizeof(_lib.PagedArgs)


class PagedCache:
    """Mixed 4/8/16-bit KV cache of many sequences, head_dim 64. Sequences are named by the ints that add(), adopt()
    and fork() return.

    max_tokens: room for that many tokens at 16 bits in full pages (some more at 8, three times as many at 4); a
    sequence's last page, and one after which the width changes, may be part full. precision as in GPUCache.
    The calls on one cache belong on one stream, or on streams that wait for each other: pages that a call frees are
    written again by later ones. Threads may call at once; what one of them frees, cuts or moves makes the others' planned
    steps refuse, as it does its own, so each holds `lock` from a step() or advance() to the last launch or replay over it.
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
        block = BLOCK * 512 * 2 * layers * heads
        if arena_bytes is None:
            arena_bytes = -(-max(max_tokens, 1) // BLOCK_TOKENS) * block
        self.arena_bytes = int(arena_bytes) // block * block
        pool = ctypes.c_void_p()
        _lib.check(_lib.load().dkv_pool_create(layers, heads, q_heads, PRECISIONS[precision], self.arena_bytes, ctypes.byref(pool)),
                   'dkv_pool_create')
        self._pool = pool.value
        # (every call holds it from its look at the pages, or at a step's generation, to its launch)
        self.lock = threading.RLock()
        at = ctypes.c_void_p()
        _lib.check(_lib.load().dkv_pool_generation(self._pool, ctypes.byref(at)), 'dkv_pool_generation')
        self._generation = ctypes.c_int64.from_address(at.value)  # counts the calls that freed, cut or moved pages
        self._length = _lib.load().dkv_pool_length
        weakref.finalize(self, _lib.load().dkv_pool_destroy, self._pool)
        with torch.inference_mode(False):
            self.arena = torch.empty(self.arena_bytes, dtype=torch.uint8, device=self.device)
        self.device = self.arena.device  # (with its index, whatever the current device is later)
        self._index = self.arena.get_device()
        self._arena_ptr = self.arena.data_ptr()

    def __reduce_ex__(self, protocol):
        raise TypeError('a PagedCache cannot be copied or pickled: fork its sequences')

    def _stream(self):
        """Torch's current stream on this cache's device."""
        return _lib.raw_stream(self._index) if self._index >= 0 else 0

    @staticmethod
    def _over(what):
        raise ValueError(f'{what}: pages were freed, cut or moved since this step was planned')

    def _launch(self, what, call, stream=None, step=None):
        """call(stream) on this cache's device and torch's current stream there, over `step` if that is given."""
        index = self._index
        if index < 0:
            raise ValueError(f'{what}: PagedCache requires a CUDA device')
        if stream is None:
            stream = _lib.raw_stream(index)
        with self.lock:
            if step is not None and step.generation != self._generation.value:
                self._over(what)
            if torch.cuda.current_device() == index:
                rc = call(stream)
            else:
                with torch.cuda.device(index):
                    rc = call(stream)
        if rc:
            _lib.check(rc, what)

    def _captured(self, stream):
        """Whether the current stream of this cache's device records a graph (the default one, 0, never does)."""
        if not stream:
            return 0
        if torch.cuda.current_device() == self._index:
            return int(torch.cuda.is_current_stream_capturing())
        with torch.cuda.device(self._index):
            return int(torch.cuda.is_current_stream_capturing())

    def _not_captured(self, what):
        if self._captured(self._stream()):
            raise ValueError(f'{what} cannot run while a graph is captured')

    # -- sequences -------------------------------------------------------------
    @staticmethod
    def _ids(seqs):
        """(array, number) of the ids of one or several sequences."""
        seqs = [seqs] if isinstance(seqs, (int, np.integer)) else list(seqs)
        ints = set(map(type, seqs)) <= {int} or all(isinstance(s, (int, np.integer)) for s in seqs)
        if not ints or seqs and not 0 <= min(seqs) <= max(seqs) < IDS:
            raise ValueError(f'sequences are named by the ints of add(), adopt() and fork(), got {seqs!r}')
        return (ctypes.c_int64 * len(seqs))(*seqs), len(seqs)

    @staticmethod
    def _whole(x, what):
        try:
            return operator.index(x)
        except TypeError:
            raise ValueError(f'{what}: {x!r} is no whole number') from None

    @staticmethod
    def _each(x, n, what):
        if isinstance(x, int):
            x = [x] * n
        elif not getattr(x, 'ndim', 1) or not hasattr(x, '__iter__'):
            x = [PagedCache._whole(x, what)] * n
        else:
            x = list(x)
            if not set(map(type, x)) <= {int}:
                x = [PagedCache._whole(v, what) for v in x]
        if len(x) != n:
            raise ValueError(f'one {what} a sequence: {len(x)} for {n}')
        for v in (min(x), max(x)) if x else ():
            if not -1 << 31 <= v < 1 << 31:
                raise ValueError(f'{what}: {v} is out of range')
        return x

    def _sequence(self, seq):
        (seq,), _ = self._ids([seq])
        out = (ctypes.c_int64 * 3)()
        at = ctypes.addressof(out)
        rc = _lib.load().dkv_pool_sequence(self._pool, seq, at, at + 8, at + 16)
        if rc:
            _lib.check(rc, 'dkv_pool_sequence')
        return out[0], out[1], out[2] & 0xffffffff

    def add(self):
        """A new, empty sequence."""
        seq = ctypes.c_int64()
        _lib.check(_lib.load().dkv_pool_add(self._pool, ctypes.byref(seq)), 'dkv_pool_add')
        return seq.value

    def length(self, seq):
        """Tokens that a sequence holds, those of steps that were planned among them."""
        if type(seq) is not int or not 0 <= seq < IDS:
            self._ids([seq])
        n = self._length(self._pool, seq)
        if n < 0:
            _lib.check(_lib.DKV_EINVAL, 'dkv_pool_length')
        return n

    def position(self, seq):
        """Position of a sequence's next token: its length and what an evicted GPUCache that it was adopted from had
        dropped."""
        length, dropped, _ = self._sequence(seq)
        return length + dropped

    def pages(self, seq):
        """A sequence's pages in token order: [(place in the arena and width as include/dkv.h names a page, tokens that
        it holds, sequences that hold it)]."""
        n = self._sequence(seq)[2]
        page, rows, holders = (ctypes.c_uint32 * n)(), (ctypes.c_int32 * n)(), (ctypes.c_int32 * n)()
        _lib.check(_lib.load().dkv_pool_pages(self._pool, seq, n, page, rows, holders), 'dkv_pool_pages')
        return list(zip(page, rows, holders))

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
        seq = ctypes.c_int64()
        self._launch('dkv_pool_adopt', lambda stream: _lib.load().dkv_pool_adopt(
            self._pool, cache.arena.data_ptr(), cache.arena.numel(), cache._tiles_host_ptr, cache._tiles_before(cache.seen[0]), cache.seen[0],
            cache.dropped, self._arena_ptr, stream, ctypes.byref(seq)))
        return seq.value

    def fork(self, seq, n=1):
        """n new sequences that go on from this one. They share its pages but a last one that is not full, of which
        each gets a copy."""
        (seq,), _ = self._ids([seq])
        n = self._whole(n, 'fork')
        if not 0 <= n <= 1 << 20:
            raise ValueError(f'fork: cannot make {n} branches')
        self._not_captured('fork')
        out = (ctypes.c_int64 * n)()
        self._launch('dkv_pool_fork', lambda stream: _lib.load().dkv_pool_fork(self._pool, seq, n, self._arena_ptr, stream, out))
        return list(out)

    def free(self, seqs):
        """Ends sequences; pages that no other one holds are free again."""
        ids, n = self._ids(seqs)
        self._not_captured('free')
        with self.lock:
            rc = _lib.load().dkv_pool_free(self._pool, ids, n)
        if rc:
            _lib.check(rc, 'dkv_pool_free')

    def truncate(self, seq, length):
        """Drops a sequence's tokens from `length` on. A cut within a page that other sequences hold copies what stays of it
        before it frees the pages behind; a cache without room for the copy refuses it, and says which cut comes first."""
        (seq,), _ = self._ids([seq])
        length = self._whole(length, 'truncate')
        if not 0 <= length < IDS:
            raise ValueError(f'truncate: a sequence cannot hold {length} tokens')
        self._not_captured('truncate')
        self._launch('dkv_pool_truncate', lambda stream: _lib.load().dkv_pool_truncate(self._pool, seq, length, self._arena_ptr, stream))

    def compact(self):
        """Brings the pages of each width together into as few blocks as hold them: what was free in pieces can hold
        pages of any width. Returns how many pages were moved. (Calls that find too little room do it themselves.)
        Steps that were planned before have to be planned again."""
        self._not_captured('compact')
        moved = ctypes.c_int64()
        self._launch('dkv_pool_compact', lambda stream: _lib.load().dkv_pool_compact(self._pool, self._arena_ptr, stream, ctypes.byref(moved)))
        return moved.value

    def _info(self):
        info = _lib.PoolInfo()
        _lib.check(_lib.load().dkv_pool_info_get(self._pool, ctypes.byref(info)), 'dkv_pool_info_get')
        return info

    def accounting(self):
        """Sequences, pages and blocks of pages by width, and bytes: of the arena, of blocks that hold pages, and of the
        pages."""
        i = self._info()
        pages = dict(zip((4, 8, 16), i.pages))
        blocks = dict(zip((4, 8, 16), i.width_blocks))
        return dict(sequences=i.sequences, pages=pages, blocks=blocks, free_blocks=i.free_blocks, allocated_bytes=self.arena_bytes,
                    block_bytes=sum(i.width_blocks) * BLOCK * i.grain,
                    page_bytes=sum(n * g for n, g in zip(i.pages, (5, 9, 16))) * i.grain)

    # -- steps -----------------------------------------------------------------
    def step(self, seqs, counts=1, bits=16, reserve=0):
        """The next tokens of some sequences: `counts` of each (one number or one a sequence), at width `bits` (too).
        Opens their pages and plans what every layer's append() and attend() do; the sequences are as long from here
        on, and what other calls read or copy of the new tokens is what append() has packed by then. The step's tensors hold the sequences' tokens one after the other, in this order. `reserve`: room in the
        plan for as many more tokens of every sequence, for steps that go on with advance(). Sequences that share
        pages attend to these together where they stand next to each other."""
        return PagedStep(self, seqs, counts, bits, reserve)

    def _check(self, what, step, layer, tensors):
        if not isinstance(step, PagedStep) or step.cache is not self:
            raise ValueError(f'{what} expects a step of this cache')
        if step.generation != self._generation.value:
            self._over(what)
        if not 0 <= layer < self.layers:
            raise ValueError(f'{what}: layer {layer} of {self.layers}')
        for x, heads in tensors:
            if x.shape != (1, heads, step.tokens, self.dim):
                raise ValueError(f'{what} expects [1, {heads}, {step.tokens}, {self.dim}], got {list(x.shape)}')
            if self._index < 0 or x.get_device() != self._index:
                raise ValueError(f'{what} requires CUDA tensors on the device of the cache')

    def append(self, k, v, layer, step):
        """Packs the step's new tokens of one layer, k and v [1, heads, tokens, 64], into their pages."""
        self._check('append', step, layer, ((k, self.heads), (v, self.heads)))
        k, kp, ks = GPUCache._rows(k)
        v, vp, vs = GPUCache._rows(v)
        stream = self._stream()
        args = _ARGS.pack(0, 0, 0, kp, ks[1], ks[2], vp, vs[1], vs[2], self._arena_ptr, self.arena_bytes, step.device_plan(stream),
                          step.plan_bytes, layer, self._captured(stream), 0.0, 0, 0, 0, 0, 0, 0, 0)
        self._launch('dkv_paged_append', lambda stream: _lib.load().dkv_paged_append(args, stream), stream, step)

    def attend(self, q, k, v, layer, step, out_dtype=None, precision=None):
        """Causal attention of the step's tokens, q [1, q_heads, tokens, 64], each over its sequence's history and the
        sequence's new tokens k, v [1, heads, tokens, 64] up to itself (these as they are, not as they are packed;
        append() may come before or after). Returns [1, tokens, q_heads, 64] in out_dtype (default q's). At precision and output
        bf16 weights have 16 bits, and are rounded to bf16 where more than 160 query rows of a KV head attend together (a prompt, or
        tokens of branches that stand next to each other, over the pages that these share); at fp32 of either 24."""
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
        stream = self._stream()
        bounds = self._captured(stream)
        need = step.workspace_bytes(bounds)
        ws = self.arena.new_empty(need) if need else None
        args = _ARGS.pack(qp, qs[1], qs[2], kp, ks[1], ks[2], vp, vs[1], vs[2], self._arena_ptr, self.arena_bytes, step.device_plan(stream),
                          step.plan_bytes, layer, bounds, self.dim ** -0.5, out.data_ptr(), self.q_heads * self.dim, self.dim,
                          out_dtype is torch.float32, PRECISIONS[precision], ws.data_ptr() if need else 0, need)
        self._launch('dkv_paged_attend', lambda stream: _lib.load().dkv_paged_attend(args, stream), stream, step)
        return out

    def materialize(self, layer, seqs, first=0, out_dtype=torch.bfloat16):
        """Dequantized tokens of one layer (None: of all), one sequence after the other: (k, v), each [1, heads,
        tokens, 64] ([layers, heads, tokens, 64]). `seqs`: sequences, of which the tokens from `first` on (one number
        or one a sequence), or a step, whose new tokens they are."""
        _check_dtype(out_dtype, 'materialize output dtype')
        if layer is not None and not 0 <= layer < self.layers:
            raise ValueError(f'materialize: layer {layer} of {self.layers}')
        self._not_captured('materialize')  # (a replay would read the pages of now)
        layer0, layers, fp32 = layer or 0, self.layers if layer is None else 1, int(out_dtype is torch.float32)
        if isinstance(seqs, PagedStep):
            self._check('materialize', seqs, 0, ())
            n, (items, n_items) = seqs.tokens, seqs.items()
        else:
            ids, count = self._ids(seqs)
            first = (ctypes.c_int64 * count)(*self._each(first, count, 'first token'))
            n = _lib.load().dkv_pool_tokens(self._pool, count, ids, first)
            if n < 0:
                _lib.check(_lib.DKV_EINVAL, 'dkv_pool_tokens')
        out = self.arena.new_empty((2, layers, self.heads, n, self.dim), dtype=out_dtype)
        if isinstance(seqs, PagedStep):
            self._launch('dkv_paged_read', lambda stream: _lib.load().dkv_paged_read(
                self._arena_ptr, self.arena_bytes, items, n_items, layer0, layers, self.layers, self.heads, out.data_ptr(), n, fp32, stream),
                step=seqs)
        else:
            self._launch('dkv_pool_read', lambda stream: _lib.load().dkv_pool_read(
                self._pool, count, ids, first, layer0, layers, self._arena_ptr, out.data_ptr(), n, fp32, stream))
        return out.unbind(0)


class PagedStep(_CacheBase):
    """The new tokens of some sequences of a PagedCache (PagedCache.step()), and what the launches over them read.

    positions: [tokens] int64 on the device, of every new token. A step can be the `past_key_values` of a decoder that
    install_packed_attention() patched: its attention then packs and attends for all the sequences. A step that a graph
    capture records can go on: advance() plans the sequences' next tokens into the same device memory, and a replay of
    the graph runs over them. (Nothing looks at a replay: once pages were freed, cut or moved, the graph is replayed after
    an advance() alone.)
    """

    backend = 'fused'
    fast_gqa = False

    def __init__(self, cache, seqs, counts, bits, reserve):
        if _CacheBase is not object:
            super().__init__()
        self.cache, self.heads, self.layers = cache, cache.heads, cache.layers
        cache._not_captured('step')
        ids, n = cache._ids(seqs)
        self.seqs = list(ids)
        self.counts, self.bits = cache._each(counts, n, 'count'), cache._each(bits, n, 'width')
        reserve = cache._whole(reserve, 'reserve')
        if not 0 <= reserve < 1 << 31:
            raise ValueError(f'step: a reserve of {reserve} tokens')
        self._ask = (n, ids, (ctypes.c_int32 * n)(*self.counts), (ctypes.c_int32 * n)(*self.bits))
        self.tokens = sum(self.counts)
        room = ctypes.c_int32()
        self._bytes = _lib.load().dkv_pool_step_bytes(cache._pool, *self._ask, reserve, ctypes.byref(room))
        if not self._bytes:
            _lib.check(_lib.DKV_EINVAL, 'dkv_pool_step_bytes')
        self._room = room.value
        with torch.inference_mode(False):
            self._dev = torch.empty(self._bytes, dtype=torch.uint8, device=cache.device)
        self._stream = _lib.raw_stream(cache.device) if cache._index >= 0 else None
        self._plan()

    def _plan(self):
        cache = self.cache
        plan, generation = _lib.PagedPlan(), ctypes.c_int64()
        with torch.inference_mode(False):
            # (pinned memory goes back to torch's cache when the copy that reads it is done)
            host = torch.empty(self._bytes, dtype=torch.uint8, pin_memory=cache._index >= 0)
        cache._launch('dkv_pool_step', lambda stream: _lib.load().dkv_pool_step(
            cache._pool, *self._ask, self._room, cache._arena_ptr, stream, host.data_ptr(), self._bytes, ctypes.byref(plan),
            ctypes.byref(generation)))
        with torch.inference_mode(False):
            self._dev.copy_(host, non_blocking=True)
        self.plan, self.plan_bytes, self.generation, self._host = plan, bytes(plan), generation.value, host
        at = 4 * plan.at_positions
        self.positions = self._dev[at:at + 8 * self.tokens].view(torch.int64)
        self._needs = {}
        if self._stream is not None:
            self.device_plan(cache._stream())  # (it was copied on the stream of now)

    def advance(self):
        """Plans the same sequences' next tokens, as many of each and at the same widths, in place of this step's. The
        launches that a capture recorded over this step run over them when they are replayed. The pages that this
        takes must fit into the room of the plan (step(..., reserve=))."""
        self.cache._not_captured('advance')
        self._plan()
        return self

    def items(self):
        """The step's rows and the pages they go to (dkv_page_rows), on the host: (address, number)."""
        return self._host.data_ptr() + 4 * self.plan.at_items, self.plan.items

    def device_plan(self, stream):
        """The plan's address, for launches on `stream`, the current one."""
        if stream != self._stream:  # (its memory is not given out again before that stream is done with it)
            self._dev.record_stream(torch.cuda.current_stream(self.cache.device))
        return self._dev.data_ptr()

    def workspace_bytes(self, bounds):
        need = self._needs.get(bounds)
        if need is None:
            args = _lib.PagedArgs(plan=self.plan, bounds=bounds)
            need = self._needs[bounds] = _lib.load().dkv_paged_workspace_bytes(ctypes.byref(args))
        return need

    # -- as the cache of a patched decoder (install_packed_attention) ------------
    def append_projection(self, qkv, cos, sin, q_heads, layer):
        """The joined Q/K/V projection [1, tokens, (q_heads + 2 heads) * 64] of one layer -> (q, k, v, 0), split, with RoPE
        from cos and sin [1, tokens, 64] and packed in one launch: what rope_qkv() and append() give, bit for bit. None
        where the inputs are not bf16 rows that the launch takes (GPUCache.append_projection)."""
        c, n = self.cache, self.tokens
        c._check('append', self, layer, ())
        if (qkv.dim() != 3 or qkv.shape[:2] != (1, n) or qkv.shape[2] != (q_heads + 2 * c.heads) * c.dim or q_heads != c.q_heads
                or cos.shape[-2:] != (n, 64) or cos.numel() != n * 64 or sin.shape != cos.shape
                or not all(t.get_device() == c._index >= 0 and t.dtype == torch.bfloat16 for t in (qkv, cos, sin))):
            return None
        qkv, cos, sin = qkv.reshape(n, -1), cos.reshape(n, 64), sin.reshape(n, 64)
        if cos.stride() != sin.stride() or any(t.stride(-1) != 1 or t.stride(0) % 8 or t.data_ptr() % 16 for t in (qkv, cos, sin)):
            return None
        q, k, v = (qkv.new_empty((1, heads, n, c.dim)) for heads in (q_heads, c.heads, c.heads))
        head, stream = n * c.dim, c._stream()
        args = _ARGS.pack(q.data_ptr(), head, c.dim, k.data_ptr(), head, c.dim, v.data_ptr(), head, c.dim, c._arena_ptr, c.arena_bytes,
                          self.device_plan(stream), self.plan_bytes, layer, c._captured(stream), 0.0, 0, 0, 0, 0, 0, 0, 0)
        c._launch('dkv_paged_rope_append', lambda stream: _lib.load().dkv_paged_rope_append(
            args, qkv.data_ptr(), qkv.stride(0), cos.data_ptr(), sin.data_ptr(), cos.stride(0), stream), stream, self)
        return q, k, v, 0

    def _fused_attention(self, n, q_heads, layer, project, cos, sin, cs_stride, qkv_out, out, stream):
        """The joined Q/K/V projection, its split and RoPE, append() and attend() for the fused decoder layer's eager
        launches, with the arguments and promises of GPUCache._fused_attention: the same bytes and outputs as the
        general entry points', which cost more host time than the GPU spends on a token of each sequence."""
        c, d = self.cache, self.cache.dim
        if n != self.tokens or q_heads != c.q_heads or layer >= c.layers:
            raise ValueError(f'a step of {self.tokens} tokens and {c.q_heads} query heads in {c.layers} layers got {n} and {q_heads} in layer {layer}')
        H, lib, here = c.heads, _lib.load(), c._stream()
        bounds = c._captured(here)
        x, x_stride, weight, w_stride, _, k, norm, eps, layout = project
        width = (q_heads + 2 * H) * d
        need = self.workspace_bytes(bounds)
        ws = c.arena.new_empty(max(need, 2 * n * width))  # (the projection's rows are done with before the attention starts)
        at, kp = ws.data_ptr(), qkv_out + q_heads * n * d * 2
        vp, head = kp + H * n * d * 2, n * d
        args = _ARGS.pack(qkv_out, head, d, kp, head, d, vp, head, d, c._arena_ptr, c.arena_bytes, self.device_plan(here), self.plan_bytes,
                          layer, bounds, d ** -0.5, out, q_heads * d, d, 0, PRECISIONS[c.precision], at if need else 0, need)
        with c.lock:
            if self.generation != c._generation.value:
                c._over('attend')
            rc = (lib.dkv_linear_tiled(x, x_stride, weight, w_stride, n, width, k, norm, eps, 0, None, 0, at, width, layout, stream)
                  or lib.dkv_paged_rope_append(args, at, width, cos, sin, cs_stride, stream) or lib.dkv_paged_attend(args, stream))
        if rc:
            _lib.check(rc, 'the launches of a fused decoder layer')

    def append(self, k, v, layer):
        self.cache.append(k, v, layer, self)
        return 0

    def attend(self, q, k, v, layer, past=0, **kw):
        return self.cache.attend(q, k, v, layer, self, **kw)

    def update(self, key_states, value_states, layer_idx, *args, **kw):
        raise ValueError('a PagedStep has no update(): its rows are read by the attention of install_packed_attention() alone')

    def _none(name):
        def refuse(self, *args, **kw):
            raise ValueError(f'a PagedStep has no {name}(): what it holds are sequences of a PagedCache')
        return refuse

    crop, reorder_cache, batch_repeat_interleave, batch_select_indices, reset = map(
        _none, ('crop', 'reorder_cache', 'batch_repeat_interleave', 'batch_select_indices', 'reset'))
    del _none

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
