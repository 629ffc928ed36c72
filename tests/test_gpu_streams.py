"""Long streams through the decoder on the GPU: what test_decoder_streams.py checks of the host, with the kernels."""
import pytest
import torch

from conftest import announce
from dkv.gpu_cache import GPUCache
from dkv.gpu_ops import sample
from dkv.streaming import StreamingDecoder, build_decoder
from test_gpu_generate import SAMPLING, inputs
from test_gpu_streaming import SMALL, frames_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('graphs', [False, True])
def test_logits_that_are_not_numbers(cuda, graphs):
    announce(f'generate from NaN logits, graphs={graphs}')
    model = build_decoder(**SMALL, seed=3)
    dec = StreamingDecoder(model, graphs=graphs)
    prefix, question, u = inputs(4)
    cache = dec.ingest(prefix, frames_for(model, 2, seed=5), [4, 8])
    norm = model.model.norm.weight  # (NaN logits; the embeddings stay)
    norm.data.fill_(float('nan'))
    assert dec.generate(cache, question, u.cuda(), **SAMPLING).tolist() == [-1] * 12
    norm.data.fill_(1.0)
    assert min(dec.generate(cache, question, u.cuda(), **SAMPLING).tolist()) >= 0


def test_forks_of_a_caller_s_cache_keep_their_rows(cuda):
    """A budgeted ingest on a cache that has a fork, over several evictions; and one on the fork itself."""
    announce('budgeted ingest on a forked cache')
    model = build_decoder(**SMALL, seed=11)
    dec = StreamingDecoder(model)
    prefix, question, u = inputs(12)
    frames, bits = frames_for(model, 20, seed=13), [4, 8, 16, 4, 8] * 4
    cache = dec.create_cache(700)
    dec.forward(cache, ids=prefix)
    fork = cache.fork()
    dec.forward(fork.fork(), ids=question)

    def rows(c):
        return [x.clone() for l in range(SMALL['layers']) for x in c.materialize(l)]
    held = rows(fork)
    out = dec.ingest(prefix[:, :1], frames, bits, cache=cache, budget=300)
    assert out is not cache and out.get_seq_length() + out.dropped == 16 + 1 + 20 * 64
    assert all(torch.equal(a, b) for a, b in zip(rows(fork), held))
    base = rows(cache)
    again = dec.ingest(prefix[:, :1], frames, bits, cache=cache.fork(), budget=300)
    assert again.get_seq_length() <= 300 and all(torch.equal(a, b) for a, b in zip(rows(cache), base))


@pytest.mark.parametrize('graphs', [False, True])
def test_a_prefix_of_half_the_budget(cuda, graphs):
    """Frames above a quarter of a budget that the prefix half fills, and a stream that goes on: eager and replayed."""
    announce(f'budget 300, prefix 150, frames of 78, graphs={graphs}')
    model = build_decoder(**SMALL, seed=11)
    frames, bits = frames_for(model, 9, seed=13, tokens=78), [4, 8, 16, 4, 8, 4, 4, 8, 16]
    g = torch.Generator().manual_seed(1)
    prefix = torch.randint(0, 512, (1, 150), generator=g)
    states = []
    for replay in {False, graphs}:
        dec = StreamingDecoder(model, graphs=replay, pipeline=1)
        for _ in range(2):
            cache = dec.ingest(prefix, frames, bits, budget=300)
            assert cache.get_seq_length() <= 300 and (cache.kept[:, :, :150] == torch.arange(150, device='cuda')).all()
            states.append([cache.kept.clone(), cache.mass().clone(), *cache.materialize(1)])
        cache = dec.ingest(prefix, frames[:4], bits[:4], cache=cache, budget=450)
        assert cache.get_seq_length() <= 450 and cache.get_seq_length() + cache.dropped == 300 + 13 * 78
    assert all(torch.equal(a, b) for state in states[1:] for a, b in zip(state, states[0]))


def test_a_cache_that_observes_goes_on_observing(cuda):
    """Frame by frame as a caller does it, over evictions by hand, and through ingests, eager and replayed."""
    announce('observing over evictions')
    model = build_decoder(**SMALL, seed=11)
    dec = StreamingDecoder(model, pipeline=1)
    prefix, question, u = inputs(12)
    frames = frames_for(model, 8, seed=13)
    cache = dec.create_cache(700)
    cache.observing = True
    dec.forward(cache, ids=prefix)
    for i, f in enumerate(frames):
        if cache.get_seq_length() > 300:
            cache = cache.evict(200, sinks=16, recent=64)
        cache.select(4, i)
        dec.forward(cache, embeddings=f)
        assert (cache.mass()[:, :, -64:] > 0).all()  # the frame's own queries were counted
    masses = []
    for graphs in (False, True, True):
        if graphs and not dec.graphs:
            dec.graphs = True
            dec.ingest(prefix, frames[:2], [4] * 2)  # (the decoder's own cache, whose captures do not count)
        own = dec._cache if graphs else dec.create_cache(700)
        own.reset()
        own.observing = True
        out = dec.ingest(prefix, frames, [4] * 8, cache=own)
        assert out is own and own.observing
        masses.append(out.mass().clone())
    assert (masses[0] > 0).all() and all(torch.equal(m, masses[0]) for m in masses[1:])


@pytest.mark.parametrize('pipeline', [1, 4])
def test_frames_replay_the_attention_that_the_cache_is_set_to(cuda, pipeline):
    """Streams that go on in the decoder's own cache, dense, then sparse over an index, then over an index that moved:
    replayed as eager."""
    announce(f'sparse frames, pipeline={pipeline}')
    model = build_decoder(**SMALL, seed=11)
    prefix, question, u = inputs(12)
    frames, bits = frames_for(model, 12, seed=13), [4, 8, 16, 4, 8, 4] * 2
    runs = []
    for graphs in (False, True):
        dec = StreamingDecoder(model, graphs=graphs, pipeline=pipeline)
        out = []
        for _ in range(2):
            cache = dec.ingest(prefix, frames, bits, qa_reserve=3000)  # (own cache with graphs: dense, captured in the first round)
            cache.index()
            cache.sparse_blocks = 2
            dec.ingest(prefix, frames, bits, cache=cache)
            cache.index()  # (longer than its buffer has room for: it moves)
            dec.ingest(prefix, frames, bits, cache=cache)
            out += [x.clone() for l in range(SMALL['layers']) for x in cache.materialize(l)]
            out.append(dec.generate(cache, question, u.cuda(), blocks=3, **SAMPLING))
            cache.sparse_blocks = 0
        runs.append(out)
    dense = StreamingDecoder(model).ingest(prefix, frames * 3, bits * 3)
    assert not torch.equal(dense.materialize(1)[0][:, :, -600:], runs[0][2][:, :, -600:])
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i


def test_positions_go_on_after_an_export_and_import(cuda):
    """An evicted cache through segments into another: the next tokens have the positions they had in the stream."""
    announce('export and import of an evicted cache')
    model = build_decoder(**SMALL, seed=14)
    dec = StreamingDecoder(model)
    prefix, question, _ = inputs(15)
    cache = dec.ingest(prefix, frames_for(model, 8, seed=16), [4, 8, 16, 4] * 2, budget=300)
    assert cache.dropped
    copy = dec.create_cache(600)
    assert copy.import_segments(cache.export_segments(), dropped=cache.dropped) == 0 and copy.dropped == cache.dropped
    want = dec.forward(cache.fork(), ids=question, logits=13)
    assert torch.equal(dec.forward(copy.fork(), ids=question, logits=13), want)
    copy.reset()
    assert copy.dropped == 0


def test_numbers_past_32_bits(cuda):
    """A top_k or a number of blocks of more than 32 bits: refused where it is negative, all of them where not."""
    announce('top_k and blocks past 32 bits')
    x, u = torch.randn(3, 100, device=cuda), torch.rand(3, device=cuda)
    for k in (-1, -(1 << 32), -(1 << 32) + 5, -(1 << 40)):
        with pytest.raises(ValueError, match='top_k'):
            sample(x, u, top_k=k)
    assert sample(x, u, top_k=(1 << 32) + 1).tolist() == sample(x, u).tolist()
    cache = GPUCache(None, layers=1, heads=1, max_tokens=200)
    rows = torch.randn(1, 1, 131, 64, device=cuda).to(torch.bfloat16)
    past = [cache.append(rows[:, :, i:i + 65], rows[:, :, i:i + 65], 0) for i in (0, 65)][1]
    cache.index()
    args = (rows[:, :, :1], rows[:, :, :1], rows[:, :, :1], 0, past)
    want = cache.attend_sparse(*args, 1000)
    for blocks in (1 << 31, 1 << 32, 10 ** 12):
        assert torch.equal(cache.attend_sparse(*args, blocks), want)
