"""evict against its definition: which tokens every layer and head keeps, their packed values and masses, the
new cache's bookkeeping, what it attends to, and that the old cache and its branches stay as they were."""
import pytest
import torch

from conftest import announce
from dkv.gpu_cache import GPUCache
from oracle.attention import attention
from test_gpu_sparse import RAGGED, build, chunk_of

pytestmark = pytest.mark.gpu

LONG = [(39, 16), (64, 4), (78, 8), (1, 4), (130, 16), (64, 8), (17, 4), (63, 8), (200, 4), (64, 16), (30, 8), (5, 16)]


def chosen(mass, segments, keep, sinks, recent):
    """[layers, heads, kept] old indices, by the definition, a layer and head at a time; the new segments."""
    starts = [sum(t for t, _ in segments[:i]) for i in range(len(segments) + 1)]
    n = starts[-1]
    a = next((i for i in range(len(segments)) if starts[i] >= sinks), len(segments))
    b = next((i for i in range(len(segments), a, -1) if starts[i] <= n - recent), a)
    if keep >= n:
        a = b = len(segments)
    middle = segments[a:b]
    total = sum(t for t, _ in middle)
    left = keep - (n - total)
    widths = list(dict.fromkeys(w for _, w in middle))
    held = {w: sum(t for t, x in middle if x == w) for w in widths}
    share = {w: left * held[w] // total for w in widths}
    for w in sorted(widths, key=lambda w: (-(left * held[w] % total), -w))[:left - sum(share.values())]:
        share[w] += 1
    new = segments[:a] + [(share[w], w) for w in widths if share[w]] + segments[b:]
    out = []
    for row in mass.flatten(0, 1).tolist():
        kept = list(range(starts[a]))
        for w in widths:
            tokens = [t for i in range(a, b) if segments[i][1] == w for t in range(starts[i], starts[i + 1])]
            tokens.sort(key=lambda t: (-row[t], t))
            kept += sorted(tokens[:share[w]])
        out.append(kept + list(range(starts[b], n)))
    return torch.tensor(out, dtype=torch.int32).view(*mass.shape[:2], -1), new


def rows_at(x, kept):
    """x [layers, heads, tokens, 64] at kept [layers, heads, k]."""
    return x.gather(2, kept.long()[..., None].expand(*kept.shape, 64))


def check(cuda, segments, heads, layers, keep, sinks, recent, into=None, mass=None, seed=0):
    announce(f'evict segments={len(segments)} heads={heads} layers={layers} keep={keep} sinks={sinks} recent={recent}')
    c, dk, dv = build(cuda, segments, heads, layers, seed)
    g = torch.Generator().manual_seed(seed + 50)
    if mass is None:  # values that repeat, so that ties are cut too
        mass = torch.randint(0, 40, (layers, heads, dk.shape[2]), generator=g).float() / 8
    c.mass().copy_(mass)
    new = c.evict(keep, sinks, recent, into=into)
    want, now = chosen(mass, segments, keep, sinks, recent)
    n = sum(t for t, _ in now)
    assert new.seen == [n] * layers and new.dropped == dk.shape[2] - n
    assert torch.equal(new.kept.cpu(), want)
    assert torch.equal(new.mass().cpu(), mass.gather(2, want.long()))
    assert new._mass[:, :, n:].abs().sum() == 0
    assert [(s.rows, s.bits) for s in new.segments] == now
    assert torch.equal(new.tiles[:len(new.tile_starts)].cpu().flatten(),
                       torch.from_numpy(new.tiles_host[:len(new.tile_starts)].copy().view('u1')).flatten())
    for l in range(layers):
        got = new.materialize(l, torch.float32)
        for x, d in zip(got, (dk, dv)):
            assert torch.equal(x[0].cpu(), rows_at(d, want)[l])
    for l in range(layers):  # the old cache holds what it held
        got = c.materialize(l, torch.float32)
        assert torch.equal(got[0][0].cpu(), dk[l]) and torch.equal(got[1][0].cpu(), dv[l])
    return c, new, (dk, dv, want)


@pytest.mark.parametrize('keep,sinks,recent', [(400, 0, 0), (400, 1, 1), (420, 39, 64), (300, 50, 99), (754, 0, 0), (1, 0, 0),
                                               (150, 39, 35), (755, 3, 3), (2000, 0, 0)])
def test_sizes_and_protected_ends(cuda, keep, sinks, recent):
    check(cuda, LONG, 3, 2, keep, sinks, recent)


@pytest.mark.parametrize('heads,layers', [(1, 1), (5, 3), (8, 1), (2, 7)])
def test_heads_and_layers(cuda, heads, layers):
    check(cuda, RAGGED, heads, layers, 333, 10, 70)


@pytest.mark.parametrize('bits', [4, 8, 16])
def test_one_width(cuda, bits):
    check(cuda, [(64, bits)] * 9 + [(33, bits)], 2, 2, 301, 64, 33)


def test_more_tokens_than_threads_and_one_row_tiles(cuda):
    check(cuda, [(1000, 4), (700, 8)] + [(1, 16)] * 300 + [(900, 4)], 2, 1, 1111, 0, 100)


def test_masses_of_every_sign_and_not_a_number(cuda):
    """Negative, infinite and equal masses order as numbers do, -0 as 0, NaN below everything."""
    n = sum(t for t, _ in RAGGED)
    mass = torch.randn(1, 2, n, generator=torch.Generator().manual_seed(4)).round(decimals=1)
    mass[0, 0, ::7], mass[0, 0, 1::7] = 0.0, -0.0
    mass[0, 1, ::11], mass[0, 1, 1::11] = float('inf'), float('-inf')
    check(cuda, RAGGED, 2, 1, 400, 0, 0, mass=mass)
    c, _, _ = build(cuda, [(200, 8)], 1)
    mass = torch.arange(200.)[None, None]
    mass[0, 0, 150:] = float('nan')
    c.mass().copy_(mass)
    assert c.evict(60).kept[0, 0].tolist() == list(range(90, 150))
    assert c.evict(160).kept[0, 0].tolist() == list(range(160))


def test_attention_and_further_eviction_over_the_new_cache(cuda):
    c, new, (dk, dv, want) = check(cuda, RAGGED, 3, 1, 400, 39, 64, into=GPUCache(None, layers=1, heads=3, max_tokens=2000))
    q, kn, vn = chunk_of(3, 9, 7, 2)
    new.select(16)
    past = new.append(kn[None].to(cuda), vn[None].to(cuda), 0)
    out = new.attend(q[None].to(cuda), kn[None].to(cuda), vn[None].to(cuda), 0, past, precision='fp32', out_dtype=torch.float32)
    k, v = (torch.cat((rows_at(x, want)[0], y.float()), 1) for x, y in ((dk, kn), (dv, vn)))
    assert (out[0].cpu().double() - attention(q, k, v, past)).abs().max() < 1e-3
    sparse = new.attend_sparse(q[None].to(cuda), kn[None].to(cuda), vn[None].to(cuda), 0, past, 3, precision='fp32',
                               out_dtype=torch.float32)  # nothing indexed yet: all of it
    assert (sparse[0].cpu().double() - attention(q, k, v, past)).abs().max() < 1e-3
    before = new.mass().clone()
    assert before[:, :, past:].abs().sum() == 0
    # back into the first cache, which is emptied
    second = new.evict(200, 39, 7, into=c)
    assert second is c and c.seen == [200] and c.dropped == sum(t for t, _ in RAGGED) - 400 + 407 - 200
    assert torch.equal(c.mass(), before.gather(2, c.kept.long()))
    assert c.frame_id == new.frame_id


def test_branches_of_the_old_cache_stay(cuda):
    c, dk, _ = build(cuda, RAGGED, 2)
    c.mass().fill_(1.)
    branch = c.fork()
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(2, 6, 4, 3))
    branch.append(kn, vn, 0)
    want = branch.attend(q, kn, vn, 0, c.seen[0])
    new = c.evict(100)
    small = branch.evict(50, recent=4)  # a branch can be evicted from
    assert torch.equal(branch.attend(q, kn, vn, 0, c.seen[0]), want)
    assert torch.equal(small.materialize(0)[0][:, :, -4:], kn)
    assert new.kept.shape == (1, 2, 100)


def test_graph_steps_of_the_new_cache_go_on(cuda):
    """A decode step captured on a cache replays over what an eviction put there."""
    into = GPUCache(None, layers=1, heads=3, max_tokens=1200)
    into.select(16)
    g = torch.Generator().manual_seed(5)
    kv = torch.randn(1, 3, 40, 64, generator=g).to(torch.bfloat16).to(cuda)
    into.append(kv, kv, 0)
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(3, 9, 1, 1))
    into.mass()
    steps = into.begin_graph_steps(1, q_heads=9)
    past = into.graph_step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        into.append(kn, vn, 0)
        into.observe(q, kn, 0, past)
        out = into.attend(q, kn, vn, 0, past)
    steps.upload()
    graph.replay()
    into.end_graph_steps()
    for keep in (300, 500):
        c, _, _ = build(cuda, RAGGED, 3)
        c.mass().copy_(torch.rand(1, 3, c.seen[0], generator=g))
        c.evict(keep, into=into)
        before = into.mass().clone()
        into.begin_graph_steps(1, steps=steps)
        past = into.graph_step()
        graph.replay()
        into.end_graph_steps()
        eager = into.attend(q, kn, vn, 0, past)
        torch.cuda.synchronize()
        assert past == keep and torch.equal(out, eager)
        mass = into.attention_mass(q, kn, 0, past)
        mass[:, :past] += before[0]
        assert torch.equal(into.mass()[0], mass)


def test_refusals(cuda):
    c, _, _ = build(cuda, RAGGED, 3)
    with pytest.raises(ValueError, match='no attention mass'):
        c.evict(100)
    c.mass()
    for kw, msg in [(dict(keep=50, sinks=39, recent=64), 'protected'), (dict(keep=-1), 'negative'), (dict(keep=1, recent=-1), 'negative'),
                    (dict(keep=100, into=c), 'this cache'), (dict(keep=100, into=c.fork()), 'branch'),
                    (dict(keep=100, into=GPUCache(None, layers=1, heads=2, max_tokens=900)), 'same layers'),
                    (dict(keep=100, into=GPUCache([(16, 700)], layers=1, heads=3)), 'online'),
                    (dict(keep=100, into=GPUCache(None, layers=1, heads=3, max_tokens=99)), 'limit')]:
        with pytest.raises(ValueError, match=msg):
            c.evict(**kw)
    planned = GPUCache([(16, 64)], layers=1, heads=1)
    with pytest.raises(ValueError, match='online'):
        planned.evict(3)
    c.begin_graph_steps(1)
    with pytest.raises(ValueError, match='graph steps'):
        c.evict(100)
    c.end_graph_steps()
    small = GPUCache(None, layers=1, heads=3, max_tokens=900, arena_bytes=256)
    assert c.evict(100, into=small) is small and small.arena_bytes > 256  # its arena grows as an append's would


def test_empty_cache(cuda):
    c = GPUCache(None, layers=2, heads=2, max_tokens=64)
    assert c.mass().shape == (2, 2, 0)
    new = c.evict(10)
    assert new.seen == [0, 0] and new.kept.shape == (2, 2, 0) and new.dropped == 0
