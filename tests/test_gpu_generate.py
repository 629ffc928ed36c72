"""Long streams through the decoder: frames within a budget, then tokens drawn from the history, dense and sparse,
eager and as graph replays."""
import pytest
import torch

from conftest import announce
from dkv.gpu_ops import sample
from dkv.streaming import StreamingDecoder, build_decoder
from test_gpu_streaming import SMALL, frames_for

pytestmark = pytest.mark.gpu

SAMPLING = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)


def inputs(seed, question=13):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 512, (1, 16), generator=g), torch.randint(0, 512, (1, question), generator=g), \
        torch.rand(12, generator=g)


def test_tokens_equal_one_forward_at_a_time(cuda):
    """generate() gives what a caller gets from forwards of its own on a fork."""
    announce('generate vs forwards')
    model = build_decoder(**SMALL, seed=3)
    dec = StreamingDecoder(model)
    prefix, question, u = inputs(4)
    cache = dec.ingest(prefix, frames_for(model, 5, seed=5), [4, 8, 16, 4, 8])
    seen = list(cache.seen)
    got = dec.generate(cache, question, u.cuda(), **SAMPLING)
    assert got.shape == (12,) and got.dtype == torch.int64 and cache.seen == seen
    branch, ids, want = cache.fork(), question, []
    for i in range(12):
        logits = dec.forward(branch, ids=ids, logits=1)[0]
        want.append(sample(logits, u[i:i + 1].cuda(), **SAMPLING))
        ids = want[-1][None]
    assert got.tolist() == torch.cat(want).tolist()
    greedy = dec.generate(cache, question, u.cuda(), temperature=0.0)
    assert greedy.tolist() == dec.generate(cache, question, 1 - u.cuda(), temperature=0.0).tolist()
    assert dec.generate(cache, question, u.cuda()[:0]).shape == (0,)
    with pytest.raises(ValueError, match='one random number'):
        dec.generate(cache, question, u.cuda()[None])


@pytest.mark.parametrize('blocks', [0, 3, 1000])
def test_replayed_tokens_equal_eager_ones(cuda, blocks):
    """The first token runs eagerly, the second is captured, the rest replay: also across requests, over a longer
    history and a renewed index."""
    announce(f'generate, graphs vs eager, blocks={blocks}')
    model = build_decoder(**SMALL, seed=3)
    dec = StreamingDecoder(model, pipeline=2)
    prefix, question, u = inputs(6)
    frames, bits = frames_for(model, 9, seed=7), [4, 8, 16, 4, 8, 4, 4, 16, 8]

    def requests():
        out = []
        for n in (6, 9, 9):
            cache = dec.ingest(prefix, frames[:n], bits[:n])
            out.append(dec.generate(cache, question, u.cuda(), blocks=blocks, **SAMPLING).tolist())
            out.append(dec.generate(cache, question, 1 - u.cuda(), blocks=blocks, temperature=1.3).tolist())
        return out

    eager = requests()
    dec.graphs = True
    assert requests() == eager
    assert len(set(map(tuple, eager))) > 2


def test_all_blocks_attend_to_all_of_the_history(cuda):
    """With as many blocks as tiles the logits are dense attention's, to the rounding of the layers."""
    model = build_decoder(**SMALL, seed=8)
    dec = StreamingDecoder(model, precision='fp32')
    prefix, question, _ = inputs(9)
    cache = dec.ingest(prefix, frames_for(model, 6, seed=10), [4, 8, 16, 4, 8, 4])
    cache.index()
    logits = []
    for blocks in (0, 100, 1):
        branch = cache.fork()
        branch.sparse_blocks = blocks
        logits.append(dec.forward(branch, ids=question, logits=question.shape[1]))
    assert (logits[0] - logits[1]).abs().max() <= 0.05  # (16-bit layers between: the bound of the native comparison)
    assert not torch.equal(logits[0], logits[2])


@pytest.mark.parametrize('pipeline', [1, 4])
def test_budgeted_ingest_replayed_equals_eager(cuda, pipeline):
    """Twenty frames within a budget of seven: what is kept, where and with what mass is the same eager and
    replayed, twice, and the history goes on to answer and to generate."""
    announce(f'budgeted ingest, pipeline={pipeline}')
    model = build_decoder(**SMALL, seed=11)
    dec = StreamingDecoder(model, pipeline=pipeline)
    prefix, question, u = inputs(12)
    bits = ([4, 8, 16, 4, 8] * 4)[:20]
    frames = frames_for(model, 20, seed=13)
    budget = 16 + 7 * 64

    def request():
        cache = dec.ingest(prefix, frames, bits, budget=budget)
        tokens = dec.generate(cache, question, u.cuda(), blocks=2, **SAMPLING).tolist()
        scores = dec.answer(cache, question, [question[:, :5], question[:, 3:9]])
        torch.cuda.synchronize()
        state = [cache.kept.clone(), cache.mass().clone()] + [x for l in range(SMALL['layers']) for x in cache.materialize(l)]
        return cache, tokens, [t.clone() for t in state + [scores]]

    cache, tokens, want = request()
    n = cache.get_seq_length()
    assert n <= budget and n + cache.dropped == 16 + 20 * 64 and not cache.observing
    assert (cache.kept[:, :, :16] == torch.arange(16, device='cuda')).all()  # the prefix
    dec.graphs = True
    for _ in range(3):
        again, same, got = request()
        assert again is dec._cache and again.plan == cache.plan and again.dropped == cache.dropped
        assert same == tokens
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # requests without a budget on the same decoder run as before
    dec.ingest(prefix, frames[:3], bits[:3])
    assert dec._cache.dropped == 0 and dec._cache.get_seq_length() == 16 + 3 * 64


def test_positions_go_on_after_an_eviction(cuda):
    """A forward after an eviction rotates its tokens by the positions they have in the stream."""
    model = build_decoder(**SMALL, seed=14)
    dec = StreamingDecoder(model)
    prefix, question, _ = inputs(15)
    cache = dec.create_cache(600)
    cache.mass()
    cache.observing = True
    dec.forward(cache, ids=prefix)
    dec.forward(cache, embeddings=frames_for(model, 4, seed=16)[0].repeat(1, 4, 1))
    new = cache.evict(100, sinks=16)
    want = dec.forward(new.fork(), ids=question, positions=torch.arange(272, 285, device='cuda'), logits=13)
    assert torch.equal(dec.forward(new.fork(), ids=question, logits=13), want)
    assert new.dropped == 172


def test_budgets_that_do_not_fit(cuda):
    model = build_decoder(**SMALL, seed=14)
    dec = StreamingDecoder(model)
    prefix, _, _ = inputs(15)
    frames = frames_for(model, 6, seed=16)
    with pytest.raises(ValueError, match='budget'):
        dec.ingest(prefix, frames, [4] * 6, budget=10)
    with pytest.raises(ValueError, match='protected|negative'):
        dec.ingest(prefix, frames, [4] * 6, budget=80)
    cache = dec.ingest(prefix, frames, [4] * 6, budget=10 ** 6)
    assert cache.dropped == 0 and cache.kept is None and (cache.mass() > 0).any()
