"""The bookkeeping of a cache after an eviction, taken over from the evicted one, is that of opening its segments."""
import random

import numpy as np
import pytest

from dkv.gpu_cache import GPUCache


def cache(lengths, bits, tokens):
    c = GPUCache(None, layers=2, heads=3, max_tokens=tokens, device='cpu')
    if lengths:
        c._open_segments(0, lengths, bits)
    c.seen = [sum(lengths)] * 2
    for i, s in enumerate(c.segments):
        s.frame = 100 + i
    return c


@pytest.mark.parametrize('seed', range(40))
def test_kept_segments_lie_as_opened_ones(seed):
    rng = random.Random(seed)
    lengths = [rng.choice([1, 1, 1, 5, 64, 65, 130, 200]) for _ in range(rng.randint(1, 30))]
    bits = [rng.choice([4, 8, 16, 16]) for _ in lengths]
    old, n = cache(lengths, bits, 8192), sum(lengths)
    sinks, recent = rng.choice([0, 0, 3, 70]), rng.choice([0, 0, 2, 90])
    ends = sum(s.rows for s in old.segments if s.start < sinks or s.end > n - recent)
    for keep in {n, n - 1, ends, (ends + n) // 2, ends + 1}:
        if keep < ends or keep < 0:
            continue
        a, b, share, held = old._eviction(keep, sinks, recent)
        into, want = cache([], [], 8192), cache([], [], 8192)
        into._open_kept(old, a, b, share)
        kept = old.segments[:a] + [None] * len(share) + old.segments[b:]
        rows = [s.rows for s in old.segments[:a]] + list(share.values()) + [s.rows for s in old.segments[b:]]
        if not rows:
            continue
        want._open_segments(0, rows, [s.bits for s in old.segments[:a]] + list(share) + [s.bits for s in old.segments[b:]])
        tiles = len(want.tile_starts)
        assert np.array_equal(into.tiles_host[:tiles], want.tiles_host[:tiles])
        for name in ('tile_starts', 'tile_singles', 'plan', 'host_counts', 'arena_used'):
            assert getattr(into, name) == getattr(want, name), name
        for x, y, z in zip(into.segments, want.segments, kept):
            assert (x.start, x.rows, x.bits, x.offset, x.tile0) == (y.start, y.rows, y.bits, y.offset, y.tile0)
            assert x.frame == (-1 if z is None else z.frame)
        assert len(into.segments) == len(want.segments)


def test_a_small_arena_grows():
    old = cache([64] * 20, [8] * 20, 4096)
    into = GPUCache(None, layers=2, heads=3, max_tokens=4096, device='cpu', arena_bytes=256)
    into._open_kept(old, *old._eviction(700, 64, 64)[:3])
    assert into.arena_used <= into.arena_bytes == into.arena.numel()
