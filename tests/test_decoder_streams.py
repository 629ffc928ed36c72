"""The decoder's host side over long streams on the CPU: caches whose launches are left out and a model that is not run."""
import types

import pytest
import torch

from dkv import _lib, streaming
from dkv.gpu_cache import GPUCache, GraphSteps
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


@pytest.mark.parametrize('budget,prefix,lengths', [
    (256, 150, [64] * 8), (300, 150, [78] * 9), (464, 16, [64] * 20), (256, 200, [20] * 30), (256, 250, [5] * 9),
    (256, 20, [100, 3, 90, 64, 1, 120, 78, 78, 200, 10]), (80, 16, [64, 8, 8, 8, 30]), (100, 60, [39] * 4), (1000, 1, [998] * 4)])
def test_budgets_that_hold_the_prefix_and_a_frame(hosted, budget, prefix, lengths):
    """Whatever the frames' lengths: the history never passes the budget, the prefix stays, and more than it."""
    left = []
    evict = GPUCache.evict

    def spy(self, keep, **kw):
        out = evict(self, keep, **kw)
        left.append((out.segments[0].rows, out.seen[0]))
        return out
    GPUCache.evict = spy
    try:
        out = hosted.ingest(prefix_of(prefix), *frames(*lengths), budget=budget)
    finally:
        GPUCache.evict = evict
    assert hosted.most <= budget and out.get_seq_length() + out.dropped == prefix + sum(lengths)
    assert left and all(first == prefix and n > prefix for first, n in left)


@pytest.mark.parametrize('budget,prefix,lengths', [
    (80, 16, [64] * 6), (100, 60, [40, 10, 40]), (256, 150, [10, 106, 10]), (300, 150, [20, 151]), (64, 64, [1])])
def test_budgets_that_do_not_are_refused_before_any_forward(hosted, budget, prefix, lengths):
    cache = hosted.create_cache(2000)
    before = state_of(cache)
    with pytest.raises(ValueError, match='budget.*protected'):
        hosted.ingest(prefix_of(prefix), *frames(*lengths), cache=cache, budget=budget)
    assert state_of(cache) == before and not hasattr(hosted, 'most') and cache._mass is None
    hosted.ingest(prefix_of(prefix), *frames(*lengths), cache=cache, budget=prefix + sum(lengths))  # (nothing is evicted)
    with pytest.raises(ValueError, match='no plan'):
        hosted.ingest(prefix_of(16), *frames(64), cache=GPUCache([(16, 300)], layers=2, heads=1, device='cpu'), budget=200)


@pytest.mark.parametrize('budget,prefix', [(300, 16), (300, 100), (200, 30)])
def test_a_stream_that_goes_on_stays_within_its_budget(hosted, budget, prefix):
    """Ingests into the cache of the one before, whose first tokens stay: also the next prefix passes no budget."""
    cache, total = None, 0
    for n in (64, 50, 64):
        cache = hosted.ingest(prefix_of(prefix), *frames(*[n] * 7), cache=cache, budget=budget, qa_reserve=100)
        total += prefix + 7 * n
        assert cache.get_seq_length() + cache.dropped == total and hosted.most <= budget
        assert cache.segments[0].rows == prefix
    with pytest.raises(ValueError, match='budget.*protected'):
        hosted.ingest(prefix_of(prefix), *frames(budget - prefix), cache=cache, budget=budget)


def test_the_newest_frames_that_leave_room_stay(hosted):
    """The last quarter of the budget, whole frames: as many of the newest as fit beside the prefix."""
    # 190 tokens, 150 of them to keep: 50 beside the prefix, one whole frame of the two in the quarter
    one = hosted.ingest(prefix_of(100), *frames(30, 30, 30, 30), budget=200)
    assert [s.rows for s in one.segments] == [100, 20, 30, 30]
    two = hosted.ingest(prefix_of(10), *frames(30, 30, 30, 30, 30, 30, 30), budget=200)
    assert [s.rows for s in two.segments] == [10, 80, 30, 30, 30]


SETTINGS = dict(observing=True, sparse_blocks=7, chunk_splits=3, as_replayed=True, chunk_segments=[0, 4, 9])


@pytest.mark.parametrize('given', [False, True])
def test_settings_go_with_an_eviction(hosted, given):
    cache, into = hosted.create_cache(300), hosted.create_cache(300) if given else None
    cache.select(8, 5)
    hosted.forward(cache, ids=prefix_of(200))
    cache.mass()
    cache.__dict__.update(SETTINGS)
    out = cache.evict(100, into=into)
    assert {k: getattr(out, k) for k in SETTINGS} == SETTINGS and (out.pending_bits, out.frame_id) == (8, 5)
    assert into is None or out is into
    again = cache.evict(300, into=into)  # (nothing leaves)
    assert again.observing and again.sparse_blocks == 7
    fork = cache.fork().evict(100)
    assert not fork.observing and fork.sparse_blocks == 7  # (a fork does not count)


@pytest.mark.parametrize('budget', [None, 300])
@pytest.mark.parametrize('observing', [False, True])
def test_an_ingest_leaves_the_settings_of_a_cache(hosted, monkeypatch, budget, observing):
    """A cache that observes goes on observing through an ingest, with and without a budget, and after it; one that
    does not observes during a budgeted one alone."""
    cache, during = hosted.create_cache(2000), []
    forward = type(hosted).forward
    monkeypatch.setattr(type(hosted), 'forward', lambda self, cache, **kw: (during.append((cache.observing, cache.sparse_blocks)),
                                                                            forward(self, cache, **kw))[1])
    cache.observing, cache.sparse_blocks = observing, 5
    out = hosted.ingest(prefix_of(16), *frames(*[64] * 12), cache=cache, budget=budget)
    assert (out is cache) == (budget is None)
    assert set(during) == {(observing or budget is not None, 5)}
    assert (out.observing, cache.observing, out.sparse_blocks, cache.sparse_blocks) == (observing, observing, 5, 5)


def test_captured_forwards_are_told_apart(monkeypatch):
    """By what a forward is captured under, and dropped where the cache holds another index or other masses."""
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda: None)
    cache, d = GPUCache(None, layers=1, heads=1, max_tokens=256, device='cpu'), decoder()
    keys = []
    for observing in (False, True):
        for blocks in (0, 3, 4):
            cache.observing, cache.sparse_blocks = observing, blocks
            keys += [d._graph_key(cache, 64), d._graph_key(cache, 64, 2)]
    assert len(set(keys)) == 12 and keys[:2] == [64, (64, 2)]

    def captured():
        steps = GraphSteps(cache, 1)
        steps.mass, steps.bounds = cache._own_mass(), cache._bounds
        return dict(steps=steps), dict(steps=[steps, GraphSteps(cache, 1)])
    one, group = captured()
    graphs = {1: one, 2: group}
    assert d._captured(graphs, 1, cache) is one and d._captured(graphs, 2, cache) is group and d._captured(graphs, 3, cache) is None
    cache._bounds = torch.zeros(16, dtype=torch.uint8)
    assert d._captured(graphs, 1, cache) is None and d._captured(graphs, 2, cache) is None and not graphs
    graphs[1], _ = captured()
    cache._mass = cache._mass.clone()
    assert d._captured(graphs, 1, cache) is None and not graphs
    graphs[1] = dict(steps=GraphSteps(cache, 1))  # (neither recorded)
    cache._bounds, cache._mass = None, None
    assert d._captured(graphs, 1, cache) is graphs[1]


def test_positions_of_imported_segments_are_checked():
    c = GPUCache(None, layers=1, heads=1, max_tokens=64, device='cpu')
    with pytest.raises(ValueError, match='dropped'):
        c.import_segments({0: []}, dropped=-1)
    c._open_segment(0, 8, 16)
    c.seen = [8]
    with pytest.raises(ValueError, match='dropped'):
        c.import_segments({0: []}, dropped=5)
    assert c.import_segments({0: []}) == 8 and c.dropped == 0


def test_blocks_past_32_bits_are_all_blocks(monkeypatch):
    """A number of blocks that no 32-bit argument holds is as many as there are, not what is left of it."""
    seen = []
    cache = GPUCache(None, layers=1, heads=1, max_tokens=64, device='cpu')
    steps = GraphSteps(cache, 1)
    room = _lib.load().dkv_attend_sparse_workspace_bytes
    monkeypatch.setattr(_lib.load(), 'dkv_attend_sparse_workspace_bytes',
                        lambda a, s: (seen.append(s._obj.blocks), room(a, s))[1])
    for blocks in (7, 1 << 32, (1 << 31) + 5):
        cache.sparse_blocks = blocks
        steps.workspace_bytes(2)
    assert seen == [7, (1 << 31) - 1, (1 << 31) - 1]


def test_an_eviction_passes_over_empty_segments():
    """An append of no tokens opens a segment of none, whose width counts for nothing."""
    c = GPUCache(None, layers=1, heads=1, max_tokens=400, device='cpu')
    at = 0
    for n, bits in [(0, 8), (64, 4), (0, 16), (64, 16), (0, 8), (64, 4), (0, 4)]:
        c._open_segment(at, n, bits)
        at += n
    c.seen = [at]
    assert c._eviction(96, 0, 0) == (0, 7, {4: 64, 16: 32}, {4: 128, 16: 64})
    assert c._eviction(96, 1, 0)[2:] == ({16: 16, 4: 16}, {16: 64, 4: 64})


def test_a_cache_smaller_than_the_budget_is_refused_before_any_forward(hosted):
    cache = hosted.create_cache(250)
    with pytest.raises(ValueError, match='budget.*250'):
        hosted.ingest(prefix_of(16), *frames(*[64] * 5), cache=cache, budget=300)
    assert not hasattr(hosted, 'most') and cache.seen == [0, 0]
    assert hosted.ingest(prefix_of(16), *frames(*[64] * 3), cache=cache, budget=300) is cache  # (never as long)
    assert hosted.ingest(prefix_of(16), *frames(*[64] * 5), cache=cache, budget=250).get_seq_length() <= 250
