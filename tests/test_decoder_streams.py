"""The decoder's host side over long streams on the CPU: caches whose launches are left out and a model that is not run."""
import types

import pytest
import torch

from dkv import streaming
from dkv.gpu_cache import GPUCache
from dkv.streaming import StreamingDecoder


class Branch:
    sparse_blocks = 0


def decoder(**kw):
    d = object.__new__(StreamingDecoder)
    d.__dict__.update(dict(graphs=False, pipeline=1, group_splits=None, precision='bf16', _cache=None, _spare=None, _graphs={},
                           _group_graphs={}, _qa_graphs={}, _qa_seen=set()), **kw)
    return d


def test_no_token_is_looked_up_where_none_could_be_drawn(monkeypatch):
    """A row without a token that can be drawn gives -1: that is never an index into the embeddings, and the tokens
    after it are -1 too."""
    drawn, looked_up = iter([5, -1, 7, -1, 2]), []

    def forward(branch, ids, logits):
        looked_up.append(ids.clone())
        return torch.zeros(1, 1, 10)
    d = decoder(_fork_forward=forward)
    monkeypatch.setattr(streaming, 'sample', lambda *a: torch.tensor([next(drawn)]))
    cache = types.SimpleNamespace(fork=Branch)
    out = d.generate(cache, torch.tensor([[3, 4]]), torch.zeros(5))
    assert out.tolist() == [5, -1, -1, -1, -1] and out.dtype == torch.int64
    assert all((ids >= 0).all() for ids in looked_up) and looked_up[1].tolist() == [[5]]


@pytest.fixture
def hosted(monkeypatch):
    """A decoder whose caches are on the CPU and whose forwards append without a launch: the host's side alone."""
    monkeypatch.setattr(GPUCache, '_call', lambda self, name, *args: None)

    class Hosted(StreamingDecoder):
        def __init__(self):
            self.__dict__.update(decoder().__dict__)
            self.text = types.SimpleNamespace()

        def create_cache(self, max_tokens):
            return GPUCache(None, layers=2, heads=1, max_tokens=max_tokens, device='cpu')

        def forward(self, cache, ids=None, embeddings=None, positions=None, logits=0):
            n = (ids if embeddings is None else embeddings).shape[1]
            if n:
                cache._open_segment(cache.seen[0], n, cache.pending_bits, cache.frame_id)
            cache.seen = [cache.seen[0] + n] * cache.layers
            self.most = max(getattr(self, 'most', 0), cache.seen[0])

    return Hosted()


def frames(*lengths):
    return [torch.zeros(1, n, 4) for n in lengths], [4, 8, 16, 4, 8][:1] * len(lengths)


def prefix_of(n):
    return torch.zeros((1, n), dtype=torch.long)


def state_of(cache):
    return list(cache.plan), list(cache.seen), cache.arena_used, cache.dropped, cache.kept, bytes(cache.tiles_host)


def test_a_caller_s_cache_is_not_evicted_into(hosted):
    """Over many evictions the cache that the caller gave, and forks of it, hold what they held at the first one."""
    cache = hosted.create_cache(400)
    before = []
    evict = GPUCache.evict

    def spy(self, *args, **kw):
        if self is cache:
            before.append(state_of(cache))
        return evict(self, *args, **kw)
    GPUCache.evict = spy
    try:
        cache.mass()
        fork = cache.fork()
        out = hosted.ingest(prefix_of(16), *frames(*[64] * 12), cache=cache, budget=300)
    finally:
        GPUCache.evict = evict
    assert out is not cache and out.get_seq_length() + out.dropped == 16 + 12 * 64 and out.get_seq_length() <= 300
    assert len(before) == 1 and state_of(cache) == before[0] and fork.seen == [0, 0] and fork.plan == []
    assert not out.observing and not cache.observing


def test_a_fork_can_be_ingested_into(hosted):
    base = hosted.create_cache(400)
    hosted.forward(base, ids=prefix_of(20))
    held = state_of(base)
    out = hosted.ingest(prefix_of(16), *frames(*[50] * 20), cache=base.fork(), budget=200)
    assert out.get_seq_length() + out.dropped == 20 + 16 + 1000 and out.get_seq_length() <= 200
    assert list(base.plan) == held[0] and base.seen == held[1]


def test_evictions_take_turns_between_two_caches(hosted, monkeypatch):
    """However many evictions: two caches of the ingest's own beside the caller's, one where it made that itself."""
    made = []
    init = GPUCache.__init__
    monkeypatch.setattr(GPUCache, '__init__', lambda self, *a, **kw: (made.append(self), init(self, *a, **kw))[1])
    hosted.ingest(prefix_of(16), *frames(*[64] * 30), budget=300)
    assert len(made) == 2
    given = hosted.create_cache(600)
    made.clear()
    hosted.ingest(prefix_of(16), *frames(*[64] * 30), cache=given, budget=300)
    assert len(made) == 2
