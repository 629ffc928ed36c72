"""The long-history calls where their kernels change over: many tiles in the index, wide and many classes of tokens,
chunks of many query rows, rows of logits by the hundred, and replays whose bounds lie on one side of such a border and
whose history on the other."""
import math
import random

import pytest
import torch

import test_gpu_evict as evicting
import test_gpu_mass as massing
import test_gpu_sample as sampling
import test_gpu_sparse as sparse
from conftest import announce
from dkv.gpu_cache import GPUCache
from dkv.gpu_ops import sample
from test_gpu_sparse import RAGGED, build, chunk_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tiles', [511, 512, 513, 1030, 2048, 2049, 2200])
def test_index_of_many_tiles(cuda, tiles):
    segments = [(3, 4), (2, 8), (1, 16), (5, 4)] * (tiles // 4) + [(2, 4)] * (tiles % 4)
    for nq, blocks in ((1, 40), (17, 7), (2, tiles - 1)):
        sparse.check(cuda, segments, 2, 6, nq, blocks, 'bf16', seed=tiles)


def capture(cuda, c, heads, q_heads, call):
    """A recorded single-token step of `call(q, k, v, past)` over an append, and a function that replays it with
    the next token."""
    q, kn, vn = (torch.zeros(1, h, 1, 64, dtype=torch.bfloat16, device=cuda) for h in (q_heads, heads, heads))
    steps = c.begin_graph_steps(1, q_heads=q_heads)
    past = c.graph_step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append(kn, vn, 0)
        out = call(q, kn, vn, past)
    steps.upload()
    graph.replay()
    c.end_graph_steps()

    def step(qi, ki, vi):
        c.begin_graph_steps(1, steps=steps)
        past = c.graph_step()
        q.copy_(qi), kn.copy_(ki), vn.copy_(vi)
        graph.replay()
        c.end_graph_steps()
        return out, past
    return step


def tokens(cuda, n, heads, q_heads, seed):
    g = torch.Generator().manual_seed(seed)
    return [tuple(torch.randn(1, h, 1, 64, generator=g).to(torch.bfloat16).to(cuda) for h in (q_heads, heads, heads))
            for _ in range(n)]


@pytest.mark.parametrize('blocks', [1, 9])
def test_replays_over_a_history_that_left_the_index(cuda, blocks):
    """The launch was recorded over an index of nearly all that the cache holds; after a reset none of the history
    is in it, and every tile of it is a unit of its own: more than the index and the tail after it once were."""
    announce(f'replay without the index, blocks={blocks}')
    c = GPUCache(None, layers=1, heads=2, max_tokens=400)
    g = torch.Generator().manual_seed(1)
    k = torch.randn(1, 2, 380, 64, generator=g).to(torch.bfloat16).to(cuda)
    c.append_batch(k, k, [4] * 380, [1] * 380)
    c.index()
    step = capture(cuda, c, 2, 6, lambda q, kn, vn, past: c.attend_sparse(q, kn, vn, 0, past, blocks))
    for n in (390, 40, 3):
        c.reset()
        c.append_batch(k[:, :, :380].repeat(1, 1, 2, 1)[:, :, :n].contiguous(), k.repeat(1, 1, 2, 1)[:, :, :n].contiguous(), [4] * n, [1] * n)
        for i, t in enumerate(tokens(cuda, 4, 2, 6, n)):
            out, past = step(*t)
            eager = c.attend_sparse(*t, 0, past, blocks)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), (n, i)
        c.index()
        out, past = step(*tokens(cuda, 1, 2, 6, 99)[0])
        assert torch.equal(out, c.attend_sparse(*tokens(cuda, 1, 2, 6, 99)[0], 0, past, blocks))


@pytest.mark.parametrize('tiles', [600, 2300])
def test_replays_whose_bounds_take_the_long_kernels(cuda, tiles):
    """Recorded over an index of many tiles, replayed over few: what a call over few gives."""
    announce(f'replay, bound of {tiles} tiles')
    c = GPUCache(None, layers=1, heads=2, max_tokens=2 * tiles)
    g = torch.Generator().manual_seed(2)
    k = torch.randn(1, 2, tiles, 64, generator=g).to(torch.bfloat16).to(cuda)
    c.append_batch(k, k, [8] * tiles, [1] * tiles)
    c.index()
    step = capture(cuda, c, 2, 6, lambda q, kn, vn, past: c.attend_sparse(q, kn, vn, 0, past, 5))
    for n in (tiles, 100, 6):
        c.reset()
        c.append_batch(k[:, :, :n].contiguous(), k[:, :, :n].contiguous(), [8] * n, [1] * n)
        c.index()
        for i, t in enumerate(tokens(cuda, 3, 2, 6, n)):
            out, past = step(*t)
            eager = c.attend_sparse(*t, 0, past, 5)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), (n, i)


@pytest.mark.parametrize('segments', [[(5000, 8)], [(64, 4)] * 210, [(13000, 4), (30, 8)], [(64, 8), (64, 4)] * 560 + [(100, 16)],
                                      [(33000, 4), (500, 16)], [(64, 16)] + [(64, 4)] * 1030 + [(1, 8)] * 40],
                         ids=['5000', '210tiles', '13000', '1121tiles', '33000', '65920'])
def test_classes_of_many_tokens(cuda, segments):
    n = sum(t for t, _ in segments)
    for keep in (n // 3, n - 1):
        evicting.check(cuda, segments, 1, 1, keep, 0, 0)


@pytest.mark.parametrize('seed', [0, 1])
def test_kept_places_become_tokens_once(cuda, seed):
    """Most of three classes of some 10000 tokens stay: every place of a kept token is read by its own thread alone
    before the token takes its place (a place read after it pointed behind the last class's tokens)."""
    frames = random.Random(seed).choices([4, 8, 16], weights=[.4, .4, .2], k=351)
    segments = [(63, 16)] + [(78, b) for b in frames] + [(35, 4)]
    n = sum(t for t, _ in segments)
    mass = torch.rand(2, 5, n, generator=torch.Generator().manual_seed(seed))
    evicting.check(cuda, segments, 5, 2, n - 587, 54, 4101, mass=mass, seed=seed)


def test_eviction_on_another_stream(cuda):
    c, _, _ = build(cuda, RAGGED, 3)
    c.mass().copy_(torch.rand(1, 3, c.seen[0], generator=torch.Generator().manual_seed(6)))
    want = c.evict(300, 39, 64)
    keys = want.materialize(0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        new = [c.evict(300, 39, 64) for _ in range(3)]
        got = [x.materialize(0) for x in new]
    torch.cuda.synchronize()
    for x, kv in zip(new, got):
        assert torch.equal(x.kept, want.kept) and all(torch.equal(a, b) for a, b in zip(kv, keys))


@pytest.mark.parametrize('nq', [30, 100, 520])
def test_observed_replays_of_many_rows(cuda, nq):
    """90, 300 and 1560 query rows a KV head: rows joined by every workgroup, once, and added up in parts."""
    announce(f'mass replay nq={nq}')
    c, _, _ = build(cuda, RAGGED, 2, extra=5 * nq)
    want = torch.zeros(2, c.capacity, device=cuda)
    c.mass()
    g = torch.Generator().manual_seed(nq)
    chunks = [tuple(torch.randn(1, h, nq, 64, generator=g).to(torch.bfloat16).to(cuda) for h in (6, 2)) for _ in range(4)]
    q, kn = (t.clone() for t in chunks[0])
    steps = c.begin_graph_steps(nq, q_heads=6)
    past = c.graph_step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append(kn, kn, 0)
        c.observe(q, kn, 0, past)
    steps.upload()
    graph.replay()
    c.end_graph_steps()
    for i, (qi, ki) in enumerate(chunks):
        if i:
            c.begin_graph_steps(nq, steps=steps)
            past = c.graph_step()
            q.copy_(qi), kn.copy_(ki)
            graph.replay()
            c.end_graph_steps()
        want[:, :past + nq] += c.attention_mass(qi, ki, 0, past)
        torch.cuda.synchronize()
        assert torch.equal(c._mass[0], want), i


@pytest.mark.parametrize('nq', [520, 700])
@pytest.mark.parametrize('precision', ['bf16', 'fp32'])
def test_mass_of_many_rows(cuda, nq, precision):
    massing.check(cuda, RAGGED, 2, 6, nq, precision)
    massing.check(cuda, RAGGED, 1, 3, nq, precision, parts=[0, 64, 65, nq - 1, nq])


@pytest.mark.parametrize('nq', [1, 5, 23, 70])
def test_mass_on_another_stream_and_keys_at_minus_infinity(cuda, nq):
    """A key that is -infinity for every query gets nothing, also where a block has rows to spare."""
    c = GPUCache(None, layers=1, heads=1, max_tokens=400)
    g = torch.Generator().manual_seed(nq)
    k = torch.randn(1, 1, 100, 64, generator=g).to(torch.bfloat16)
    k[0, 0, 40] = -math.inf
    q, kn = torch.rand(1, 3, nq, 64, generator=g).to(torch.bfloat16) + 0.125, torch.randn(1, 1, nq, 64, generator=g).to(torch.bfloat16)
    c.append(k.to(cuda), k.to(cuda), 0)
    dense = torch.cat((k, kn), 2)[0].float()
    dense[0, 40] = 0
    s = q[0].double() @ dense.double().transpose(1, 2) / 8
    mask = torch.ones(nq, 100 + nq, dtype=torch.bool).tril(100)
    mask[:, 40] = False
    ref = torch.softmax(s.masked_fill(~mask, -math.inf), -1).sum((0, 1))[None]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = c.attention_mass(q.to(cuda), kn.to(cuda), 0, 100)
    torch.cuda.synchronize()
    assert out[0, 40] == 0
    massing.check_close(out, ref)


def test_hundreds_of_rows_with_parameters_of_their_own(cuda):
    """More rows than are handled at a time, some with a short list, some with none."""
    n = 700
    x, u = sampling.rows_of(n, 331, torch.bfloat16, 30)
    g = torch.Generator().manual_seed(31)
    pick = lambda *values: torch.tensor(values)[torch.randint(0, len(values), (n,), generator=g)]
    t, p, m = pick(0.5, 1.0, 0.0, 1.5), pick(1.0, 0.5, 0.75), pick(0.0, 0.0, 0.0625)
    k = pick(0, 3, 40, 256, 257, 300, 400).int()
    announce('sample 700 rows of mixed parameters')
    out = sample(x.to(cuda), u.to(cuda), t.to(cuda), k.to(cuda), p.to(cuda), m.to(cuda)).tolist()
    assert out == [sampling.drawn(x[i], u[i].double().item(), t[i].item(), int(k[i]), p[i].item(), m[i].item()) for i in range(n)]
    for kw in (dict(), dict(top_p=0.5), dict(top_k=30), dict(top_k=300, min_p=0.0625)):
        sampling.check(cuda, x, u, **kw)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('kw', [dict(top_k=257, top_p=0.9), dict(top_k=9000, top_p=0.3), dict(top_k=256, top_p=0.99),
                                dict(top_k=40000, top_p=0.97, min_p=1e-4), dict(top_k=5000, min_p=0.2)],
                         ids=lambda kw: '-'.join(f'{k}{v}' for k, v in kw.items()))
def test_many_kept_of_a_large_vocabulary(cuda, kw, dtype):
    sampling.check(cuda, *sampling.rows_of(2, 49281, dtype, 32), **kw)


def test_vocabularies_past_half_a_million(cuda):
    """Parts too long for the registers of a workgroup, and the longest row there is."""
    x, u = sampling.rows_of(1, 600011, torch.float32, 50)
    for kw in (dict(top_k=20), dict(top_p=0.9), dict(temperature=0.0)):
        sampling.check(cuda, x, u, **kw)
    x = torch.full((1, 1 << 22), -math.inf, dtype=torch.bfloat16, device=cuda)
    x[0, 4000000] = x[0, 7] = 1.0
    for v, want in ((0.25, 7), (0.75, 4000000)):
        assert sample(x, torch.tensor([v], device=cuda), top_p=0.99).tolist() == [want]
    with pytest.raises(ValueError, match='vocab'):
        sample(torch.zeros(1, (1 << 22) + 1, device=cuda), u.to(cuda))


def test_keeping_nothing_empties_the_cache(cuda):
    c, _, _ = build(cuda, RAGGED, 2)
    c.mass()
    new = c.evict(0)
    assert new.seen == [0] and new.kept.shape == (1, 2, 0) and new.dropped == c.seen[0]
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(2, 6, 3, 8))
    assert new.append(kn, vn, 0) == 0
    out = new.attend_sparse(q, kn, vn, 0, 0, 4, out_dtype=torch.float32)
    ref = sparse.expected(q[0].cpu(), kn[0].float().cpu(), vn[0].float().cpu(), 0, torch.zeros(2, 3, 0, dtype=torch.bool))
    assert ((out[0].cpu().double() - ref).abs() <= sparse.tolerance(ref, vn.cpu(), torch.float32, 'bf16')).all()


def test_token_strides_at_their_border(cuda):
    """A chunk's rows up to 2^23 - 8 elements apart are read where they lie; a larger stride is refused, but of one row."""
    c, dk, dv = build(cuda, RAGGED, 1)
    c.index()
    past = c.seen[0]
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(1, 3, 2, 9))
    want, mass = c.attend_sparse(q, kn, vn, 0, past, 3), c.attention_mass(q, kn, 0, past)
    for stride in ((1 << 23) - 8, 1 << 23):
        far = torch.zeros(2 * stride, dtype=torch.bfloat16, device=cuda).as_strided((1, 1, 2, 64), (0, 0, stride, 1))
        for x in (kn, vn):
            far.copy_(x)
            k, v = (far, vn) if x is kn else (kn, far)
            if stride < 1 << 23:
                assert torch.equal(c.attend_sparse(q, k, v, 0, past, 3), want)
                assert torch.equal(c.attention_mass(q, k, 0, past), mass)
            else:
                with pytest.raises(ValueError, match='token stride'):
                    c.attend_sparse(q, k, v, 0, past, 3)
        one = c.attend_sparse(q[:, :, :1], far[:, :, :1], vn[:, :, :1], 0, past, 3)
        assert torch.equal(one, c.attend_sparse(q[:, :, :1], vn[:, :, :1], vn[:, :, :1], 0, past, 3))
    with pytest.raises(ValueError, match='token stride'):
        c.attention_mass(q, far, 0, past)


def test_two_streams_draw_at_once(cuda):
    rows = [sampling.rows_of(4, 49280, torch.bfloat16, 40 + i) for i in range(4)]
    rows = [(x.to(cuda), u.to(cuda)) for x, u in rows]
    want = [sample(x, u, top_p=0.9) for x, u in rows]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, (x, u) in enumerate(rows * 3):
        with torch.cuda.stream(sides[i % 2]):
            got.append(sample(x, u, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want * 3))
