"""Workspace of sparse attention: what its scores take, and that scoring a range of queries at a time changes nothing."""
import ctypes

import pytest
import torch

from conftest import announce
from dkv import _lib
from dkv.gpu_cache import GPUCache


def room(nq, heads, tiles, blocks, group=1):
    a, s = _lib.AttnArgs(), _lib.Sparse(None, tiles, blocks, 0, 0)
    a.nq, a.heads, a.q_heads, a.layers, a.n_tiles, a.past = nq, heads, heads * group, 1, tiles, tiles * 64
    return _lib.load().dkv_attend_sparse_workspace_bytes(ctypes.byref(a), ctypes.byref(s))


def test_scores_take_room_only_where_they_are_written():
    """An index of up to 512 tiles is scored and chosen from in one launch, which keeps the scores."""
    lists = 4 * 8 * 2048 * 16
    assert room(2048, 8, 512, 16) == lists
    assert room(512, 8, 513, 16) == 4 * 8 * 512 * 513 + 4 * 8 * 512 * 16
    assert room(2048, 8, 512, 512) == room(2048, 8, 2000, 2000) == 0  # nothing to choose


@pytest.mark.parametrize('nq,heads,tiles', [(65535, 8, 2048), (65535, 32, 8192), (40000, 5, 100000), (17, 8, 1 << 24)])
def test_scores_of_many_queries_over_a_long_index_take_a_bounded_room(nq, heads, tiles):
    row = 4 * heads * tiles
    lists = 4 * heads * nq * 16
    # few queries are split over up to 1024 workgroups, which leave 64 values, a maximum and a sum of one query head each:
    # 264 bytes; four pieces are rounded up to 256 bytes
    assert room(nq, heads, tiles, 16) - lists <= max(64 << 20, 16 * row) + 1024 * 264 + 4 * 256
    assert room(1, heads, tiles, 16) >= row + 4 * heads * 16


@pytest.mark.gpu
@pytest.mark.parametrize('nq', [1904, 1905, 2000, 3900])
def test_queries_scored_in_ranges_choose_as_in_one(cuda, nq):
    """8 KV heads over 1100 indexed tiles: 1904 queries at a time. The first four heads alone are scored in one or two
    other ranges."""
    announce(f'sparse, {nq} queries over 1100 tiles')
    g = torch.Generator().manual_seed(nq)
    tiles, H = 1100, 8
    k, v = (torch.randn(1, H, 4 * tiles + nq, 64, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
    q = torch.randn(1, 2 * H, nq, 64, generator=g).to(torch.bfloat16).to(cuda)
    outs = []
    for heads in (H, 4, 1):
        cache = GPUCache(None, layers=1, heads=heads, max_tokens=4 * tiles + nq, precision='bf16')
        cache.append_batch(k[:, :heads, :4 * tiles], v[:, :heads, :4 * tiles], [8, 4] * (tiles // 2), [4] * tiles)
        assert cache.index() == tiles
        outs.append(cache.attend_sparse(q[:, :2 * heads], k[:, :heads, 4 * tiles:], v[:, :heads, 4 * tiles:], 0, 4 * tiles, 3,
                                        out_dtype=torch.float32))
    assert torch.isfinite(outs[0]).all()
    assert torch.equal(outs[0][:, :, :8], outs[1]) and torch.equal(outs[0][:, :, :2], outs[2])
