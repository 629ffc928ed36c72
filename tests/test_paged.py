"""PagedCache bookkeeping, plans and refusals on the CPU (device='cpu' arenas; no kernel runs)."""
import copy
import ctypes
import pickle
import random
import threading

import numpy as np
import pytest
import torch

from dkv import GPUCache, PagedCache, _lib
from test_long_history import test_struct_layout_matches_header as check_layout

GRAINS, PER_BLOCK = {4: 5, 8: 9, 16: 16}, {4: 9, 8: 5, 16: 3}


class Quiet(PagedCache):
    """Bookkeeping alone: what would be launched is not."""
    def __init__(self, *a, **kw):
        super().__init__(*a, device='cpu', **kw)
        self._arena_ptr = None

    def _launch(self, what, call, stream=None):
        _lib.check(call(None), what)


def check(c, seqs):
    """Pages lie in blocks of their width, do not overlap and are held by as many sequences as name them."""
    held, info = {}, c.accounting()
    for s in seqs:
        pages = c.pages(s)
        assert sum(r for _, r, _ in pages) == c.length(s) and all(1 <= r <= 64 for _, r, _ in pages)
        assert not pages or pages[-1][1] == 64 or pages[-1][2] == 1
        for page, _, holders in pages:
            held.setdefault(page, [holders, 0])[1] += 1
    assert all(a == b for a, b in held.values())
    spans = sorted(((p >> 2), (p >> 2) + GRAINS[4 << (p & 3)], 4 << (p & 3)) for p in held)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    assert all(a // 48 == (b - 1) // 48 and a % 48 % GRAINS[w] == 0 for a, b, w in spans)
    widths = {}
    for a, _, w in spans:
        assert widths.setdefault(a // 48, w) == w
    assert info['pages'] == {w: sum(x == w for _, _, x in spans) for w in GRAINS}
    assert info['blocks'] == {w: sum(x == w for x in widths.values()) for w in GRAINS}
    assert info['free_blocks'] == info['allocated_bytes'] // (48 * c._info().grain) - len(widths)


def rows(c, seq):
    return [r for _, r, _ in c.pages(seq)]


@pytest.mark.parametrize('cls,cname', [(_lib.PagedBatch, 'dkv_paged_batch'), (_lib.PagedPlan, 'dkv_paged_plan'),
                                       (_lib.PagedArgs, 'dkv_paged_args'), (_lib.PoolInfo, 'dkv_pool_info')])
def test_struct_layout_matches_header(tmp_path, cls, cname):
    check_layout(tmp_path, cls, cname)


def test_geometry():
    c = Quiet(2, 3, 3, max_tokens=64 * 30)
    i = c._info()
    assert i.blocks == i.free_blocks == 10 and i.grain == 512 * 2 * 2 * 3 == _lib.load().dkv_page_grain(2, 3)
    for w in GRAINS:
        assert GRAINS[w] * i.grain == _lib.slab_bytes(64, w, 2, 3)
    assert c.arena_bytes == 10 * 48 * i.grain


def test_growing_fills_the_last_page_of_the_same_width_first():
    c = Quiet(1, 1, 1)
    a, b = c.add(), c.add()
    s = c.step([a, b], [70, 10], [4, 16])
    assert s.positions.tolist() == list(range(70)) + list(range(10)) and s.tokens == 80
    c.step([a, b], [60, 200], [4, 16])
    c.step([a], [1], [8])
    s = c.step(a, 1, 4)
    assert s.positions.tolist() == [131]
    assert rows(c, a) == [64, 64, 2, 1, 1] and c.length(a) == 132
    assert rows(c, b) == [64, 64, 64, 18]
    assert [4 << (p & 3) for p, _, _ in c.pages(a)] == [4, 4, 4, 8, 4]
    check(c, [a, b])


def test_a_full_cache_refuses_and_stays_as_it_was():
    c = Quiet(1, 1, 1, max_tokens=64 * 6)  # 2 blocks
    a, b = c.add(), c.add()
    c.step(a, 64 * 4 + 63)
    before = (c.accounting(), c.pages(a))
    for seqs, counts, bits in ((a, 66, 16), (a, 1, 4), ([b, a], [1, 65], [16, 16]), ([a, b], [1, 1], [16, 8])):
        with pytest.raises(ValueError, match='full'):
            c.step(seqs, counts, bits)
        assert (c.accounting(), c.pages(a)) == before and c.length(b) == 0
    with pytest.raises(ValueError, match='full'):
        c.fork(a, 2)
    with pytest.raises(ValueError, match='1'):
        c.fork(a, -1)
    assert (c.accounting(), c.pages(a)) == before
    (d,) = c.fork(a)
    with pytest.raises(ValueError, match='full'):
        c.truncate(d, 10)  # a page that both hold: a copy has no room
    assert c.length(d) == 64 * 4 + 63
    check(c, [a, b, d])


def test_branches_share_full_pages_and_copy_a_part_one():
    c = Quiet(1, 1, 1)
    a = c.add()
    c.step(a, 130, 8)
    b, d = c.fork(a, 2)
    assert c.pages(b)[:2] == c.pages(a)[:2] and c.pages(a)[0][2] == 3
    assert len({c.pages(s)[2][0] for s in (a, b, d)}) == 3
    check(c, [a, b, d])
    c.free(a)
    check(c, [b, d])
    c.truncate(b, 100)  # into a page that d holds too
    assert rows(c, b) == [64, 36] and rows(c, d) == [64, 64, 2] and c.pages(b)[1][0] != c.pages(d)[1][0]
    check(c, [b, d])
    c.truncate(b, 64)
    c.truncate(b, 0)
    assert c.pages(b) == []
    seqs = [b, d] + c.fork(b, 1) + c.fork(d, 0) + c.fork(d, 5)
    check(c, seqs)
    c.free(seqs)
    assert c.accounting()['page_bytes'] == 0


def test_compacting_leaves_as_few_blocks_as_hold_the_pages():
    c = Quiet(1, 1, 1, max_tokens=64 * 300)
    seqs = [c.add() for _ in range(40)]
    for i in range(4):
        for j, s in enumerate(seqs):
            c.step(s, 64, (4, 8, 16)[(i + j) % 3])
    c.free(seqs[::2])
    left, old = seqs[1::2], {s: c.pages(s) for s in seqs[1::2]}
    moved = c.compact()
    assert moved == sum(a != b for s in left for a, b in zip(old[s], c.pages(s))) > 0
    for s in left:
        assert [(p & 3, r) for p, r, _ in old[s]] == [(p & 3, r) for p, r, _ in c.pages(s)]
    info = c.accounting()
    assert all(info['blocks'][w] == -(-info['pages'][w] // PER_BLOCK[w]) for w in GRAINS)
    check(c, left)
    assert c.compact() == 0


def test_room_in_pieces_is_brought_together():
    c = Quiet(1, 1, 1, max_tokens=64 * 6)  # 2 blocks
    a, b = c.add(), c.add()
    c.step(a, 64 * 9, 4)
    c.step(b, 64, 4)
    c.truncate(a, 64 * 3)
    step = c.step(a, 1, 4)
    c.step(b, 64, 16)  # the second block's page moves to the first
    assert c.accounting()['blocks'] == {4: 1, 8: 0, 16: 1}
    check(c, [a, b])
    with pytest.raises(ValueError, match='moved'):
        c._check('attend', step, 0, ())


def test_random_bookkeeping():
    rng = np.random.default_rng(1)
    c = Quiet(1, 2, 2, max_tokens=64 * 60)
    seqs, want = [c.add()], {0: 0}
    for _ in range(600):
        kind = rng.choice(['add', 'step', 'step', 'step', 'fork', 'free', 'truncate', 'compact'])
        some = [seqs[i] for i in rng.permutation(len(seqs))[:rng.integers(1, len(seqs) + 1)]]
        try:
            if kind == 'add':
                seqs.append(c.add())
                want[seqs[-1]] = 0
            elif kind == 'step':
                counts = rng.choice([1, 2, 63, 64, 65, 200], len(some)).tolist()
                c.step(some, counts, rng.choice([4, 8, 16], len(some)).tolist(), int(rng.integers(0, 100)))
                for s, n in zip(some, counts):
                    want[s] += n
            elif kind == 'fork':
                made = c.fork(some[0], int(rng.integers(0, 4)))
                seqs += made
                want.update((s, want[some[0]]) for s in made)
            elif kind == 'free' and len(some) < len(seqs):
                c.free(some)
                seqs = [s for s in seqs if s not in some]
            elif kind == 'truncate':
                n = int(rng.integers(0, want[some[0]] + 1))
                c.truncate(some[0], n)
                want[some[0]] = n
            elif kind == 'compact':
                c.compact()
        except ValueError as e:
            assert 'full' in str(e)
            c.free(seqs[1:])
            seqs = seqs[:1]
        check(c, seqs)
        assert all(c.length(s) == want[s] for s in seqs)


def test_calls_of_several_threads():
    """Threads that add, grow, fork, cut and end sequences of their own in one cache, and bring pages together."""
    c, errors, kept = Quiet(1, 1, 1, max_tokens=64 * 400), [], []

    def work(seed):
        try:
            rng = random.Random(seed)
            mine = [c.add()]
            for _ in range(200):
                kind, s = rng.choice(['step', 'step', 'fork', 'free', 'cut', 'compact']), rng.choice(mine)
                if kind == 'step':
                    n = c.length(s)
                    c.step(s, rng.randint(1, 100), rng.choice([4, 8, 16]))
                    assert c.length(s) > n
                elif kind == 'fork' and len(mine) < 6:
                    mine += c.fork(s, 2)
                    assert c.length(mine[-1]) == c.length(s)
                elif kind == 'free' and len(mine) > 1:
                    mine.remove(s)
                    c.free(s)
                elif kind == 'cut':
                    c.truncate(s, rng.randint(0, c.length(s)))
                elif kind == 'compact':
                    c.compact()
                if c.length(mine[0]) > 1500:
                    c.truncate(mine[0], 10)
                for x in mine[1:]:
                    if c.length(x) > 1500:
                        c.truncate(x, 20)
            kept.append(mine)
        except Exception as e:  # (an assertion too)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    check(c, [s for mine in kept for s in mine])
    c.free([s for mine in kept for s in mine])
    assert c.accounting()['page_bytes'] == 0


def test_steps_that_go_on():
    c = Quiet(1, 1, 1)
    a, b = c.add(), c.add()
    step = c.step([a, b], [3, 1], [16, 4], reserve=130)
    dev = step._dev
    for i in range(1, 44):
        step.advance()
        assert step.positions.tolist() == [3 * i, 3 * i + 1, 3 * i + 2, i] and step._dev is dev
    lengths = (c.length(a), c.length(b))
    with pytest.raises(ValueError, match='room'):
        for _ in range(400):
            step.advance()
    assert lengths[0] < c.length(a) == 3 * c.length(b)  # whole steps alone


def test_refusals():
    for kw in (dict(dim=128), dict(precision='fp8'), dict(q_heads=4), dict(layers=0), dict(arena_bytes=100), dict(layers=40000)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=1, heads=3, q_heads=3, device='cpu', arena_bytes=None), **kw})
    c = Quiet(1, 3, 6)
    a, b = c.add(), c.add()
    for call in (lambda: c.length(7), lambda: c.length(-1), lambda: c.length('a'), lambda: c.length(1 << 64), lambda: c.free([a, a]),
                 lambda: c.free([a, 9]), lambda: c.truncate(a, 1), lambda: c.truncate(a, -1), lambda: c.truncate(a, 1 << 64), lambda: c.fork(9),
                 lambda: c.fork(a, -1), lambda: c.fork(a, 1 << 32), lambda: c.step([a, a]), lambda: c.step([a], [1, 2]), lambda: c.step([a], 0),
                 lambda: c.step([]), lambda: c.step([a], 1, 5), lambda: c.step([a], 1, [4, 8]), lambda: c.step([a], 1, 16, -1),
                 lambda: c.step([a], (1 << 32) + 1), lambda: c.step([a, 5]), lambda: c.pages(5),
                 lambda: c.adopt(c), lambda: c.adopt(GPUCache(None, layers=2, heads=3, device='cpu')),
                 lambda: c.materialize(1, [a]), lambda: c.materialize(0, [a], 1), lambda: c.materialize(0, [a], -1),
                 lambda: c.materialize(0, [a], [0, 0]), lambda: c.materialize(0, [a, a]),
                 lambda: c.materialize(0, [a], out_dtype=torch.float16), lambda: c.append(None, None, 0, None)):
        with pytest.raises(ValueError):
            call()
    assert c.length(a) == c.length(b) == 0 and c.accounting()['sequences'] == 2
    x = torch.zeros(1, 3, 1, 64)
    step = c.step([a])
    for call in (lambda: c.append(x, x, 0, step), lambda: c.append(x, x, 1, step), lambda: c.append(x[:, :2], x, 0, step),
                 lambda: c.attend(x, x, x, 0, step), lambda: c.attend(x.repeat(1, 2, 1, 1), x, x, 0, step),
                 lambda: c.attend(x, x, x, 0, step, precision='half'), lambda: Quiet(1, 3, 6).append(x, x, 0, step)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError, match='CUDA'):
        c = PagedCache(1, 1, 1, device='cpu')
        c.step(c.add())


def test_caches_are_not_copied():
    c = Quiet(1, 1, 1)
    step = c.step(c.add())
    for call, x in ((copy.copy, c), (copy.deepcopy, c), (pickle.dumps, c), (copy.deepcopy, step), (pickle.dumps, step)):
        with pytest.raises(TypeError, match='copied'):
            call(x)


def test_pools_refuse_null_and_foreign_tables():
    lib = _lib.load()
    assert lib.dkv_pool_add(None, None) == _lib.DKV_EINVAL
    pool, one = Quiet(1, 1, 1), (ctypes.c_int64 * 1)(0)
    one[0] = pool.add()
    null = dict(add=(None,), info_get=(None,), generation=(None,), sequence=(0, None, None, None), compact=(None, None, None),
                fork=(one[0], 1, None, None, None), free=(None, 1), adopt=(None, 0, None, 0, 0, 0, None, None, None),
                read=(1, one, None, 0, 1, None, None, 0, 0, None), pages=(one[0], 1, None, None, None))
    for name, rest in null.items():
        assert getattr(lib, f'dkv_pool_{name}')(pool._pool, *rest) == _lib.DKV_EINVAL and b'null' in lib.dkv_last_error(), name
    assert lib.dkv_pool_tokens(pool._pool, 1, one, None) == lib.dkv_pool_length(pool._pool, 77) == -1
    assert lib.dkv_pool_step_bytes(pool._pool, 1, one, None, None, 0, None) == 0 and pool.accounting()['sequences'] == 1
    assert lib.dkv_pool_create(1, 1, 1, 0, 1 << 20, None) == _lib.DKV_EINVAL
    c = Quiet(1, 1, 1)
    tile = np.zeros(2, dtype=[('offset', '<i8'), ('start', '<i4'), ('rows', '<u2'), ('bits', 'u1'), ('pad', 'u1')])
    seq = ctypes.c_int64()
    def adopt(tokens, size=1 << 20, **kw):
        tile['offset'], tile['start'], tile['rows'], tile['bits'] = (0, 4096), (0, 10), 10, 16
        for name, x in kw.items():
            tile[name] = x
        return lib.dkv_pool_adopt(c._pool, 4096, size, tile.ctypes.data, 2, tokens, 0, None, None, ctypes.byref(seq))
    for bad in (dict(tokens=21), dict(tokens=10), dict(tokens=-1), dict(tokens=20, start=(0, 11)), dict(tokens=20, bits=(16, 5)),
                dict(tokens=20, offset=(0, 1 << 20)), dict(tokens=20, offset=(-16, 4096)), dict(tokens=20, offset=(8, 4096)),
                dict(tokens=20, rows=(10, 65)), dict(tokens=20, rows=(0, 10)), dict(tokens=20, size=4096)):
        assert adopt(**bad) == _lib.DKV_EINVAL, bad
    assert c.accounting()['sequences'] == 0
    assert adopt(15) == 0 and c.length(seq.value) == 15 and rows(c, seq.value) == [15]


def batch(count, past, pages, rows, first, heads=2, q_heads=6, layers=1, arena=1 << 20, max_pages=64, position=None, precision=0):
    arrays = [np.array(x, dtype=t) for x, t in ((count, np.int32), (past, np.int32), (position or past, np.int32), (first, np.int32),
                                                (pages, np.uint32), (rows, np.int32))]
    b = _lib.PagedBatch(len(count), *[x.ctypes.data for x in arrays], layers, heads, q_heads, arena, max_pages, precision)
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
            mine = [(int(x) * 16 << 2 | int(x) % 3) for x in ((list(range(shared)) if old else []) + (100 + 40 * i + np.arange(40)).tolist())]
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
        words, plan = write(batch(count, past, pages, rows, first, q_heads=2 * G, arena=1 << 26, max_pages=len(pages), precision=trial % 2))
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
            for f, n4, n8, pg, tok, cnt, blk, u0, u1, part, _, _ in records(at, k, 12):
                assert [held[f + u][0] & 3 for u in range(pg)] == [0] * n4 + [1] * (n8 - n4) + [2] * (pg - n8)
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
               dict(pages=[2 | 2047 << 2]), dict(q_heads=5), dict(precision=2), dict(heads=0), dict(layers=0), dict(count=[1 << 23], rows=[64])):
        with pytest.raises(ValueError):
            write(batch(**{**ok, **kw}))
    # a launch has fewer than 2^32 threads: a wave for each query row and head that is joined
    for heads, tokens, fits in ((1, 1 << 22, True), (16, 1 << 21, True), (64, 1 << 20, False), (16, 1 << 22, False)):
        b = batch([tokens], [0], [], [], [0, 0], heads=heads, q_heads=heads)
        assert (_lib.load().dkv_paged_plan_bytes(ctypes.byref(b)) > 0) == fits
        assert fits or b'too many for one step' in _lib.load().dkv_last_error()
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
                                dict(plan_words=None), dict(layer=1), dict(layer=-1), dict(plan=_lib.PagedPlan()), dict(arena_bytes=(1 << 20) - 1)])
def test_append_and_attend_refuse(kw):
    lib = _lib.load()
    for call in (lib.dkv_paged_append, lib.dkv_paged_attend):
        assert call(ctypes.byref(args(**kw)), None) == _lib.DKV_EINVAL and lib.dkv_last_error()


@pytest.mark.parametrize('kw', [dict(q=0), dict(q=4104), dict(q_tok_stride=4), dict(out=None), dict(out=4100), dict(out_tok_stride=2),
                                dict(out_dtype=2), dict(precision=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')), dict(kn_tok_stride=1 << 23), dict(vn_tok_stride=-64)])
def test_attend_refuses(kw):
    assert _lib.load().dkv_paged_attend(ctypes.byref(args(**kw)), None) == _lib.DKV_EINVAL


def test_rope_append_refuses():
    lib = _lib.load()
    for kw, qkv, row, cos, sin, cs in ((dict(layer=1), 4096, 640, 4096, 4096, 64), (dict(q=0), 4096, 640, 4096, 4096, 64),
                                       (dict(q=4104), 4096, 640, 4096, 4096, 64), (dict(q_tok_stride=4), 4096, 640, 4096, 4096, 64),
                                       ({}, None, 640, 4096, 4096, 64), ({}, 4098, 640, 4096, 4096, 64), ({}, 4096, 644, 4096, 4096, 64),
                                       ({}, 4096, 640, None, 4096, 64), ({}, 4096, 640, 4096, 4104, 64), ({}, 4096, 640, 4096, 4096, 66)):
        assert lib.dkv_paged_rope_append(ctypes.byref(args(**kw)), qkv, row, cos, sin, cs, None) == _lib.DKV_EINVAL and lib.dkv_last_error()
    assert lib.dkv_paged_rope_append(None, 4096, 640, 4096, 4096, 64, None) == _lib.DKV_EINVAL


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
    dtype = np.dtype([('src', '<i8'), ('dst', '<i8'), ('src_rows', 'u1'), ('src_row', 'u1'), ('dst_row', 'u1'), ('rows', 'u1'),
                      ('bits', 'u1'), ('reserved', 'u1', 3)])
    lib = _lib.load()
    grain = 512 * 2 * 2 * 2
    def move(*moves, src=4096, dst=4096, size=40 * grain):
        m = np.array([x + ((0, 0, 0),) for x in moves], dtype=dtype)
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
