"""A PagedCache's calls in several threads on one stream: pages that one of them frees, cuts or moves between another's look at them and
its launch."""
import threading

import pytest
import torch

from conftest import announce
from dkv import PagedCache
from dkv.streaming import StreamingDecoder, build_decoder
from test_gpu_generate import SAMPLING
from test_gpu_paged import rows_like
from test_gpu_paged_streams import streams
from test_gpu_streaming import SMALL

pytestmark = pytest.mark.gpu


def test_a_step_is_looked_at_where_it_is_launched(cuda):
    """A sequence is freed behind a call's own checks, as another thread would."""
    announce('freed before the launch')
    cache = PagedCache(1, 1, 3, max_tokens=4096)
    seq = cache.add()
    gen = torch.Generator().manual_seed(1)
    q, k = rows_like(gen, 1, 3, 5).cuda(), rows_like(gen, 1, 1, 5).cuda()
    qkv, cos = rows_like(gen, 1, 5, 5).flatten(2).cuda(), torch.ones(1, 5, 64, dtype=torch.bfloat16, device='cuda')
    launch = PagedCache._launch
    for call in (lambda s: cache.append(k, k, 0, s), lambda s: cache.attend(q, k, k, 0, s), lambda s: cache.materialize(0, s),
                 lambda s: s.append_projection(qkv, cos, cos, 3, 0)):
        other, step = cache.add(), cache.step(seq, 5)
        call(step)
        other_step = cache.step(seq, 5)

        def late(what, f, *a, **kw):
            del cache._launch
            cache.free(other)
            return launch(cache, what, f, *a, **kw)
        cache._launch = late
        with pytest.raises(ValueError, match='since this step was planned'):
            call(other_step)


def test_reads_beside_threads_that_move_pages(cuda):
    """One thread reads a sequence while others on the same stream grow, free and bring together pages around it."""
    announce('reads beside moves')
    cache = PagedCache(2, 2, 2, max_tokens=64 * 60)
    gen = torch.Generator().manual_seed(2)
    rows = rows_like(gen, 1, 2, 400).cuda()
    kept, errors, stop = cache.add(), [], threading.Event()

    def grow(seq, n, bits):
        with cache.lock:  # (a plan and the launches over it)
            step = cache.step(seq, n, bits)
            for layer in range(2):
                cache.append(rows[:, :, :n], rows[:, :, :n], layer, step)
    first = cache.add()
    grow(first, 300, 16)
    grow(kept, 400, 16)  # behind pages that come and go
    want = rows[0, :, :400]

    def churn(seq):
        try:
            for i in range(60):
                cache.free(seq)
                seq = cache.add()
                grow(seq, (100, 250, 30)[i % 3], (4, 8, 16)[i % 3])
                cache.compact()
        except Exception as e:
            errors.append(e)
        finally:
            stop.set()

    def read():
        try:
            while not stop.is_set():
                k, v = cache.materialize(None, kept)
                if not (torch.equal(k[0], want) and torch.equal(v[1], want)):
                    errors.append('rows of another sequence')
                    return
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=churn, args=(first,)), threading.Thread(target=read)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_questions_of_two_threads(cuda):
    """Two threads' generate_batch on one cache: the tokens that each gives alone."""
    announce('generate_batch of two threads')
    dec = StreamingDecoder(build_decoder(**SMALL, seed=5))
    caches, questions, u = streams(dec, 6)
    pages = dec.create_paged_cache(1 << 13)
    a, b = (pages.adopt(c) for c in caches)
    jobs = [([a, a, b, a, a], u), ([b, a, a, b, b], 1 - u)]
    alone = [dec.generate_batch(pages, s, questions, x, **SAMPLING).tolist() for s, x in jobs]
    got, errors = [None, None], []

    def work(i):
        try:
            for _ in range(3):
                got[i] = dec.generate_batch(pages, jobs[i][0], questions, jobs[i][1], **SAMPLING).tolist()
                assert got[i] == alone[i]
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert got == alone
