"""Many questions at once through the decoder: histories that ingest() packed, adopted into the pages of a PagedCache, branches of
them, prompts of all lengths in one forward and a token of each in the next ones, eager and as graph replays."""
import pytest
import torch

from conftest import announce
from dkv.gpu_ops import sample
from dkv.streaming import StreamingDecoder, build_decoder
from test_gpu_generate import SAMPLING
from test_gpu_streaming import SMALL, frames_for

pytestmark = pytest.mark.gpu


def streams(dec, seed):
    """Two ingested histories and questions of different lengths."""
    gen = torch.Generator().manual_seed(seed)
    prefix = torch.randint(0, 512, (1, 16), generator=gen)
    caches = []
    for n, tokens in ((6, 64), (3, 50)):
        frames = frames_for(dec.model, n, seed + n, tokens)
        caches.append(dec.ingest(prefix, frames, [4, 8, 16, 4, 8, 4][:n], cache=dec.create_cache(1024)))
    questions = [torch.randint(0, 512, (1, n), generator=gen) for n in (13, 1, 40, 7, 70)]
    return caches, questions, torch.rand(5, 24, generator=gen).cuda()


@pytest.mark.parametrize('fused', [True, False])
def test_a_step_of_all_questions_is_one_forward_of_each(cuda, fused):
    """Logits of ragged prompts and of the tokens after them, against a forward of each question on a fork of its GPUCache:
    within the bound of two attention kernels over the same rows in this decoder (0.05)."""
    announce(f'ragged forwards, fused={fused}')
    dec = StreamingDecoder(build_decoder(**SMALL, seed=3), fused_ops=fused, precision='fp32')
    caches, questions, _ = streams(dec, 4)
    pages = dec.create_paged_cache(1 << 13)
    a, b = (pages.adopt(c) for c in caches)
    turns = [questions, [torch.tensor([[7 * i]]) for i in range(5)], [torch.tensor([[i]]) for i in range(5)]]
    branches, got = pages.fork(a, 3) + pages.fork(b, 2), []
    for ids in turns:
        counts = [x.shape[1] for x in ids]
        step = pages.step(branches, counts)
        with torch.inference_mode():
            got.append(dec._paged_forward(step, torch.cat(ids, 1).cuda(), torch.tensor(counts).cumsum(0).sub(1).cuda()))
    for i, cache in enumerate([caches[0]] * 3 + [caches[1]] * 2):  # (forks of one cache run one after another)
        fork = cache.fork()
        for turn, ids in enumerate(turns):
            want = dec.forward(fork, ids=ids[i], logits=1)[0, 0]
            err = (got[turn][i] - want).abs().max().item()
            assert err <= 0.05, (turn, i, err)
    assert [pages.length(s) for s in (a, b)] == [c.get_seq_length() for c in caches]


def test_tokens_equal_own_forwards_and_replays(cuda):
    """generate_batch() gives what steps of a caller's own give, replayed the same tokens, and leaves the pages as they were."""
    announce('generate_batch')
    dec = StreamingDecoder(build_decoder(**SMALL, seed=5))
    caches, questions, u = streams(dec, 6)
    pages = dec.create_paged_cache(1 << 13)
    a, b = (pages.adopt(c) for c in caches)
    seqs, before = [a, a, b, a, a], pages.accounting()
    got = dec.generate_batch(pages, seqs, questions, u, **SAMPLING)
    assert got.shape == (5, 24) and got.dtype == torch.int64 and pages.accounting() == before
    branches = pages.fork(a, 2) + pages.fork(b) + pages.fork(a, 2)
    ids, want = questions, []
    for i in range(24):
        counts = [x.shape[1] for x in ids]
        step = pages.step(branches, counts)
        with torch.inference_mode():
            logits = dec._paged_forward(step, torch.cat([x.cuda() for x in ids], 1), torch.tensor(counts).cumsum(0).sub(1).cuda())
        want.append(sample(logits, u[:, i], **SAMPLING))
        ids = [x.reshape(1, 1) for x in want[-1]]
    assert got.tolist() == torch.stack(want, 1).tolist()
    pages.free(branches)
    dec.graphs = True
    for _ in range(2):
        assert dec.generate_batch(pages, seqs, questions, u, **SAMPLING).tolist() == got.tolist()
    other = dec.generate_batch(pages, a, questions, 1 - u, temperature=1.3)
    dec.graphs = False
    assert dec.generate_batch(pages, a, questions, 1 - u, temperature=1.3).tolist() == other.tolist() != got.tolist()
    for n in (0, 1, 2, 17):
        assert dec.generate_batch(pages, seqs, questions, u[:, :n], **SAMPLING).tolist() == got[:, :n].tolist()
    assert pages.accounting() == before


def test_evicted_stream_keeps_its_positions(cuda):
    """A budgeted stream's history goes on at the positions it had."""
    announce('evicted stream')
    dec = StreamingDecoder(build_decoder(**SMALL, seed=7), precision='fp32')
    gen = torch.Generator().manual_seed(8)
    prefix, question = torch.randint(0, 512, (1, 16), generator=gen), torch.randint(0, 512, (1, 21), generator=gen)
    cache = dec.ingest(prefix, frames_for(dec.model, 10, 9), [4, 8] * 5, budget=16 + 5 * 64)
    assert cache.dropped
    pages = dec.create_paged_cache(1 << 12)
    seq = pages.adopt(cache)
    step = pages.step(pages.fork(seq), 21)
    assert step.positions.tolist() == list(range(16 + 640, 16 + 640 + 21))
    with torch.inference_mode():
        got = dec._paged_forward(step, question.cuda(), slice(-1, None))
    want = dec.forward(cache.fork(), ids=question, logits=1)[0]
    assert (got - want).abs().max() <= 0.05
