"""PagedCache bookkeeping, plans and refusals on the CPU (device='cpu' arenas; no kernel runs)."""
import ctypes

import numpy as np
import pytest
import torch

from dkv import GPUCache, PagedCache, _lib
from dkv.paged_cache import BLOCK, GRAINS, PER_BLOCK


class Quiet(PagedCache):
    """Notes the moves that it would launch."""
    def __init__(self, *a, **kw):
        super().__init__(*a, device='cpu', **kw)
        self.moved = []

    def _move(self, source, moves):
        self.moved += moves


def grow(cache, seqs, counts, bits):
    cache._grow(seqs, counts, bits)


def test_pages_do_not_overlap_and_fill_blocks():
    c = Quiet(2, 3, 3, max_tokens=64 * 30)
    assert c.blocks == 10 and c.grain == 512 * 2 * 2 * 3 == _lib.load().dkv_page_grain(2, 3)
    for w in GRAINS:
        assert GRAINS[w] * c.grain == _lib.slab_bytes(64, w, 2, 3)
    taken = [c._take(w) for w in (4, 8, 16) * 5]
    spans = sorted(((p >> 2), (p >> 2) + GRAINS[4 << (p & 3)]) for p in taken)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    assert all(a // BLOCK == (b - 1) // BLOCK for a, b in spans)
    assert c._n_blocks == {4: 1, 8: 1, 16: 2}
    for p in taken:
        c._give(p)
    assert sorted(c._empty) == list(range(10)) and c._n_pages == {4: 0, 8: 0, 16: 0}


def test_growing_fills_the_last_page_of_the_same_width_first():
    c = Quiet(1, 1, 1)
    a, b = c.add(), c.add()
    grow(c, [a, b], [70, 10], [4, 16])
    grow(c, [a, b], [60, 200], [4, 16])
    grow(c, [a], [1], [8])
    grow(c, [a], [1], [4])
    assert c._seqs[a].rows.tolist() == [64, 64, 2, 1, 1] and c.length(a) == 132
    assert c._seqs[b].rows.tolist() == [64, 64, 64, 18]
    assert [4 << int(p & 3) for p in c._seqs[a].pages] == [4, 4, 4, 8, 4]


def test_a_full_cache_refuses_and_stays_as_it_was():
    c = Quiet(1, 1, 1, max_tokens=64 * 6)  # 2 blocks
    a = c.add()
    grow(c, [a], [64 * 5], [16])
    before = (c._n_pages.copy(), c._n_blocks.copy(), c.length(a))
    with pytest.raises(ValueError, match='full'):
        grow(c, [a], [65], [16])
    with pytest.raises(ValueError, match='full'):
        grow(c, [a], [1], [4])
    assert (c._n_pages, c._n_blocks, c.length(a)) == before
    grow(c, [a], [64], [16])


def test_branches_share_full_pages_and_copy_a_part_one():
    c = Quiet(1, 1, 1)
    a = c.add()
    grow(c, [a], [130], [8])
    b, d = c.fork(a, 2)
    assert c._seqs[b].pages[:2].tolist() == c._seqs[a].pages[:2].tolist()
    assert len({int(c._seqs[s].pages[2]) for s in (a, b, d)}) == 3
    assert [m[5] for m in c.moved] == [2, 2] and c._n_pages[8] == 5
    c.free(a)
    assert c._n_pages[8] == 4 and c.length(b) == 130
    c.truncate(b, 100)  # into a page that d holds too
    assert c._seqs[b].rows.tolist() == [64, 36] and c._n_pages[8] == 4
    assert c.moved[-1][5] == 36 and int(c._seqs[b].pages[1]) != int(c._seqs[d].pages[1])
    c.truncate(b, 64)
    c.truncate(b, 0)
    assert len(c._seqs[b].pages) == 0 and c._n_pages[8] == 3
    assert c.fork(b, 1) and c.fork(d, 0) == []


def test_compacting_leaves_as_few_blocks_as_hold_the_pages():
    c = Quiet(1, 1, 1, max_tokens=64 * 300)
    seqs = [c.add() for _ in range(40)]
    for i in range(4):
        for j, s in enumerate(seqs):
            grow(c, [s], [64], [(4, 8, 16)[(i + j) % 3]])
    c.free(seqs[::2])
    held = {s: (c._seqs[s].pages.copy(), c._seqs[s].rows.copy()) for s in seqs[1::2]}
    n = c.compact()
    assert n == len(c.moved) > 0
    to = {(m[0], m[6]): m[1] for m in c.moved}
    assert len(set(m[1] for m in c.moved)) == n and not set(m[0] for m in c.moved) & set(m[1] for m in c.moved)
    for s, (pages, rows) in held.items():
        for old, new in zip(pages.tolist(), c._seqs[s].pages.tolist()):
            w = 4 << (old & 3)
            assert (new >> 2) * c.grain == to.get(((old >> 2) * c.grain, w), (old >> 2) * c.grain) and old & 3 == new & 3
        assert c._seqs[s].rows.tolist() == rows.tolist()
    for w in GRAINS:
        assert c._n_blocks[w] == -(-c._n_pages[w] // PER_BLOCK[w])
    assert sum(c._n_blocks.values()) + len(c._empty) == c.blocks
    assert c.compact() == 0


def test_room_in_pieces_is_brought_together():
    c = Quiet(1, 1, 1, max_tokens=64 * 6)  # 2 blocks
    a, b = c.add(), c.add()
    grow(c, [a], [64 * 9], [4])
    grow(c, [b], [64], [4])
    c.truncate(a, 64 * 3)
    grow(c, [b], [64], [16])  # the second block's page moves to the first
    assert c.moved and c._n_blocks == {4: 1, 8: 0, 16: 1}


def test_refusals():
    for kw in (dict(dim=128), dict(precision='fp8'), dict(q_heads=4), dict(layers=0), dict(arena_bytes=100)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=1, heads=3, q_heads=3, device='cpu'), **kw})
    c = Quiet(1, 3, 6)
    a, b = c.add(), c.add()
    for call in (lambda: c.length(7), lambda: c.free([a, a]), lambda: c.free([a, 9]), lambda: c.truncate(a, 1), lambda: c.truncate(a, -1),
                 lambda: c.fork(a, -1), lambda: c.step([a, a]), lambda: c.step([a], [1, 2]), lambda: c.step([a], 0), lambda: c.step([]),
                 lambda: c.step([a], 1, 5), lambda: c.step([a], 1, [4, 8]), lambda: c.step([a], 1, 16, -1), lambda: c.step([a]),
                 lambda: c.adopt(c), lambda: c.adopt(GPUCache(None, layers=2, heads=3, device='cpu')),
                 lambda: c.materialize(1, [a]), lambda: c.materialize(0, [a], 1), lambda: c.materialize(0, [a], [0, 0]),
                 lambda: c.materialize(0, [a], out_dtype=torch.float16), lambda: c.append(None, None, 0, None)):
        with pytest.raises(ValueError):
            call()
    assert c.length(a) == c.length(b) == 0 and len(c._seqs) == 2


def batch(count, past, pages, rows, first, heads=2, q_heads=6, layers=1, arena=1 << 20, max_pages=64, position=None):
    arrays = [np.array(x, dtype=t) for x, t in ((count, np.int32), (past, np.int32), (position or past, np.int32), (first, np.int32),
                                                (pages, np.uint32), (rows, np.int32))]
    b = _lib.PagedBatch(len(count), *[x.ctypes.data for x in arrays], layers, heads, q_heads, arena, max_pages)
    b.keep = arrays
    return b


def write(b):
    lib = _lib.load()
    need = lib.dkv_paged_plan_bytes(ctypes.byref(b))
    words = np.zeros(max(need // 4, 4), dtype=np.int32)
    plan = _lib.PagedPlan()
    rc = lib.dkv_paged_plan_write(ctypes.byref(b), words.ctypes.data, need, ctypes.byref(plan))
    _lib.check(rc, 'dkv_paged_plan_write')
    return words, plan


def test_a_plan_covers_every_row_and_unit_once():
    rng = np.random.default_rng(0)
    for trial in range(60):
        n, G = int(rng.integers(1, 12)), int(rng.choice([1, 3, 8, 20]))
        count = rng.integers(1, rng.choice([2, 20, 300]), n).tolist()
        pages, rows, first, past, shared = [], [], [0], [], rng.integers(0, 12)
        for i in range(n):
            old = int(rng.integers(0, 20)) if rng.random() < .8 else 0
            mine = [(int(x) * 16 << 2 | 2) for x in ((list(range(shared)) if old else []) + (100 + 40 * i + np.arange(40)).tolist())]
            held = [64] * int(shared if old else 0)
            held += [int(x) for x in rng.integers(1, 65, old)]
            past.append(sum(held))
            left = count[i]
            if held:
                add = min(left, 64 - held[-1])
                held[-1] += add
                left -= add
            while left:
                held.append(min(left, 64))
                left -= held[-1]
            pages += mine[:len(held)]
            rows += held
            first.append(len(pages))
        words, plan = write(batch(count, past, pages, rows, first, q_heads=2 * G, arena=1 << 26, max_pages=len(pages)))
        assert plan.tokens == sum(count) and plan.work <= plan.max_work and plan.merges <= plan.max_merges
        assert plan.rows <= plan.max_rows and plan.items <= plan.max_items and plan.long_work <= plan.max_long
        def records(at, k, width):
            return words[at:at + k * width].reshape(-1, width).tolist()
        # every new row goes to one row of a page
        new = sorted((t + j, page, r + j) for t, page, r, m in records(plan.at_items, plan.items, 4) for j in range(m))
        assert [t for t, _, _ in new] == list(range(plan.tokens)) and len({(p, r) for _, p, r in new}) == len(new)
        held = records(plan.at_pages, first[-1], 2)
        # what every (token, query head) attends to: pages and new tokens, each once
        seen = {}
        parts = {}
        for at, k, block_rows in ((plan.at_work, plan.work, 16), (plan.at_long, plan.long_work, 256)):
            for f, pg, tok, cnt, blk, u0, u1, part in records(at, k, 8):
                for r in range(block_rows * blk, min(block_rows * (blk + 1), cnt * G)):
                    row = (tok + r // G, r % G)
                    units = seen.setdefault(row, [])
                    units += [('page', *held[f + u]) for u in range(u0, min(u1, pg))]
                    units += [('new', tok + 64 * (u - pg)) for u in range(max(u0, pg), u1)]
                    parts.setdefault(row, []).append(part + r - block_rows * blk if part >= 0 else -1)
        at = 0
        for i in range(n):
            at_page, have = first[i], 0
            want = []
            while have < past[i]:
                want.append(('page', pages[at_page], min(rows[at_page], past[i] - have)))
                have += rows[at_page]
                at_page += 1
            for t in range(count[i]):
                for g in range(G):
                    got = seen.pop((at + t, g))
                    new = {u for u in got if u[0] == 'new'}
                    assert sorted(u for u in got if u[0] == 'page') == sorted(want)
                    assert {('new', at + j) for j in range(0, t + 1, 64)} <= new <= {('new', at + j) for j in range(0, count[i], 64)}
                    assert len(got) == len(want) + len(new)
            at += count[i]
        assert not seen
        joined = {}
        for tok, total, r0, part, stride, shared_part, shared_stride, splits in records(plan.at_merges, plan.merges, 8):
            for r in range(r0, min(r0 + 16, total)):
                joined[(tok + r // G, r % G)] = [part + s * stride + r - r0 for s in range(splits & 0xffff)] + \
                    [shared_part + s * shared_stride + r - r0 for s in range(splits >> 16)]
        flat = [x for row, some in parts.items() for x in some if x >= 0]
        assert len(set(flat)) == len(flat) and all(x < plan.rows for x in flat)
        for row, some in parts.items():
            assert some == [-1] if row not in joined else sorted(joined[row]) == sorted(some)


def test_plans_refuse_what_the_kernels_would_trust():
    ok = dict(count=[2], past=[3], pages=[0], rows=[5], first=[0, 1])
    words, plan = write(batch(**ok, position=[10]))
    assert words[plan.at_positions:plan.at_positions + 4].view(np.int64).tolist() == [10, 11]
    grain = 512 * 2 * 2
    for kw in (dict(count=[0]), dict(past=[-1]), dict(rows=[4]), dict(rows=[6]), dict(rows=[65]), dict(pages=[3]), dict(first=[0, 0]),
               dict(first=[1, 0]), dict(max_pages=0), dict(arena=4 * grain), dict(pages=[(1 << 20) // grain << 2]),
               dict(pages=[2 | 2047 << 2]), dict(q_heads=5), dict(heads=0), dict(layers=0), dict(count=[1 << 23], rows=[64])):
        with pytest.raises(ValueError):
            write(batch(**{**ok, **kw}))
    lib = _lib.load()
    b = batch(**ok)
    assert lib.dkv_paged_plan_write(ctypes.byref(b), None, 1 << 20, ctypes.byref(plan)) == _lib.DKV_EINVAL
    words = np.zeros(64, dtype=np.int32)
    assert lib.dkv_paged_plan_write(ctypes.byref(b), words.ctypes.data, 256, ctypes.byref(plan)) == _lib.DKV_EINVAL


def args(**kw):
    _, plan = write(batch([2], [3], [0], [5], [0, 1]))
    a = _lib.PagedArgs(q=4096, q_head_stride=128, q_tok_stride=64, k_new=4096, kn_head_stride=128, kn_tok_stride=64, v_new=4096,
                       vn_head_stride=128, vn_tok_stride=64, arena=4096, arena_bytes=1 << 20, plan_words=4096, plan=plan, scale=.125,
                       out=4096, out_tok_stride=384, out_head_stride=64)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize('kw', [dict(k_new=0), dict(v_new=8), dict(kn_tok_stride=63), dict(vn_head_stride=4), dict(arena=None),
                                dict(plan_words=None), dict(layer=1), dict(layer=-1), dict(plan=_lib.PagedPlan())])
def test_append_and_attend_refuse(kw):
    lib = _lib.load()
    for call in (lib.dkv_paged_append, lib.dkv_paged_attend):
        assert call(ctypes.byref(args(**kw)), None) == _lib.DKV_EINVAL and lib.dkv_last_error()


@pytest.mark.parametrize('kw', [dict(q=0), dict(q=4104), dict(q_tok_stride=4), dict(out=None), dict(out=4100), dict(out_tok_stride=2),
                                dict(out_dtype=2), dict(precision=2), dict(kn_tok_stride=1 << 23), dict(vn_tok_stride=-64)])
def test_attend_refuses(kw):
    assert _lib.load().dkv_paged_attend(ctypes.byref(args(**kw)), None) == _lib.DKV_EINVAL


def test_attend_wants_its_workspace():
    pages = [16 * i << 2 | 2 for i in range(400)]
    _, plan = write(batch([1], [64 * 399], pages, [64] * 399 + [1], [0, 400], arena=1 << 26, max_pages=400))
    lib, a = _lib.load(), args(plan=plan)
    need = lib.dkv_paged_workspace_bytes(ctypes.byref(a))
    assert need > 0
    for workspace, size in ((None, need), (4096, need - 1), (4104, need)):
        a.workspace, a.workspace_bytes = workspace, size
        assert lib.dkv_paged_attend(ctypes.byref(a), None) == _lib.DKV_EINVAL


def test_reads_refuse_rows_outside():
    lib = _lib.load()
    def read(token=0, page=0, row0=0, rows=4, layer0=0, n_layers=1, dtype=0, arena=4096, n=8):
        items = np.array([token, page, row0, rows], dtype=np.int32)
        return lib.dkv_paged_read(arena, 1 << 20, items.ctypes.data, 1, layer0, n_layers, 2, 2, 4096, n, dtype, None)
    for kw in (dict(token=5), dict(token=-1), dict(page=3), dict(page=1 << 20), dict(row0=61), dict(row0=-1), dict(rows=0), dict(rows=65),
               dict(layer0=2), dict(n_layers=3), dict(dtype=2), dict(arena=None)):
        assert read(**kw) == _lib.DKV_EINVAL, kw


def test_moves_refuse_what_meets():
    from dkv.paged_cache import MOVE_DTYPE
    lib = _lib.load()
    grain = 512 * 2 * 2 * 2
    def move(*moves, src=4096, dst=4096, size=40 * grain):
        m = np.array([x + (0,) * 0 + ((0, 0, 0),) for x in moves], dtype=MOVE_DTYPE)
        return lib.dkv_paged_move(src, size, dst, size, m.ctypes.data, len(m), 2, 2, None)
    ok = (0, 5 * grain, 64, 0, 0, 64, 4)
    for bad in ([(0, 36 * grain, 64, 0, 0, 64, 4)], [(-16, 0, 64, 0, 0, 1, 4)], [(8, 5 * grain, 64, 0, 0, 1, 4)], [(0, 5 * grain, 64, 0, 1, 64, 4)],
                [(0, 5 * grain, 32, 10, 0, 30, 4)], [(0, 5 * grain, 64, 0, 0, 0, 4)], [(0, 5 * grain, 64, 0, 0, 1, 5)],
                [(0, 5 * grain, 65, 0, 0, 1, 4)],
                [(0, 0, 64, 0, 0, 1, 4)], [(0, 3 * grain, 64, 0, 0, 1, 4)], [ok, (10 * grain, 5 * grain, 64, 0, 63, 1, 4)],
                [ok, (5 * grain, 10 * grain, 64, 0, 0, 1, 4)], [ok, (20 * grain, 5 * grain, 64, 0, 0, 1, 8)],
                [ok, (20 * grain, 9 * grain, 64, 0, 0, 1, 4)]):
        assert move(*bad) == _lib.DKV_EINVAL, bad
    assert move(ok, src=None) == _lib.DKV_EINVAL
