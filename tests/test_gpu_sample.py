"""sample against its definition in 64 bits, token for token: every filter alone and together, ties, borders,
rows that cannot be drawn from, odd vocabularies and strides, parameters per row, and the drawn frequencies."""
import math

import pytest
import torch

from conftest import announce
from dkv.gpu_ops import sample

pytestmark = pytest.mark.gpu


def drawn(x, u, temperature, top_k, top_p, min_p):
    """The definition, a row at a time, on the CPU: weights in 64 bits, then whole multiples of 2^-200, so that every
    sum and comparison is exact."""
    x = [v if v == v else -math.inf for v in x.double().tolist()]
    top = max(x)
    if top == -math.inf:
        return -1
    if temperature == 0:
        return x.index(top)
    w = [1.0 if v == top else 0.0 if top == math.inf or v == -math.inf else math.exp((v - top) / temperature) for v in x]
    unit = [int(math.ldexp(v, 200)) for v in w]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if top_k:
        order = order[:top_k]
    if top_p < 1:
        part, whole = top_p.as_integer_ratio()
        total, kept, before = sum(unit[i] for i in order), [], 0
        for i in order:
            if kept and not before * whole < part * total:
                break
            kept.append(i)
            before += unit[i]
        order = kept
    order = sorted(i for i in order if w[i] >= min_p)
    part, whole = u.as_integer_ratio()
    total, before = sum(unit[i] for i in order), 0
    for i in order:
        before += unit[i]
        if before * whole > part * total:
            return i
    return max(i for i in order if unit[i])


def check(cuda, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    announce(f'sample {tuple(logits.shape)} {logits.dtype} T={temperature} k={top_k} p={top_p} m={min_p}')
    out = sample(logits.to(cuda), u.to(cuda), temperature, top_k, top_p, min_p)
    assert out.dtype == torch.int64 and out.shape == u.shape
    want = [drawn(x, v, temperature, top_k, top_p, min_p) for x, v in zip(logits, u.double().tolist())]
    assert out.tolist() == want
    return out


def rows_of(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype), torch.rand(rows, generator=g)


FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_p=0.5), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0),
           dict(top_k=40, top_p=0.9), dict(top_p=0.8, min_p=0.02), dict(top_k=100, top_p=0.95, min_p=0.01),
           dict(top_k=10 ** 6), dict(top_p=1e-6), dict(temperature=0.0), dict(temperature=0.2), dict(temperature=3.0, top_p=0.7)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('kw', FILTERS, ids=lambda kw: '-'.join(f'{k}{v}' for k, v in kw.items()) or 'none')
@pytest.mark.parametrize('vocab', [1, 2, 63, 1000, 5003])
def test_filters(cuda, vocab, kw, dtype):
    check(cuda, *rows_of(5, vocab, dtype, vocab), **kw)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('kw', [dict(), dict(top_k=50, top_p=0.95), dict(top_k=3000), dict(top_p=0.9, min_p=0.002)],
                         ids=['none', 'top_k-top_p', 'large_top_k', 'top_p-min_p'])
def test_large_vocabularies(cuda, kw, dtype):
    check(cuda, *rows_of(2, 49280, dtype, 1), **kw)
    check(cuda, *rows_of(1, 131071, dtype, 2), **kw)


def test_very_large_vocabulary_and_many_rows(cuda):
    check(cuda, *rows_of(1, 300007, torch.float32, 3), top_p=0.9)
    check(cuda, *rows_of(300, 257, torch.bfloat16, 4), top_k=20, top_p=0.9)


@pytest.mark.parametrize('kw', [dict(), dict(top_k=5), dict(top_p=0.5), dict(top_k=6, top_p=0.5), dict(min_p=1.0)],
                         ids=lambda kw: '-'.join(kw) or 'none')
def test_equal_logits(cuda, kw):
    """All tokens tie: the filters cut them by index, and borders fall on exact multiples."""
    n = 1000
    x = torch.zeros(9, n)
    u = torch.tensor([0.0, 0.25, 0.5, 0.499999, 0.75, 0.125, 0.999, 1 - 2.0 ** -24, 0.6])
    check(cuda, x, u, **kw)
    x[:, ::3] = -1.0
    check(cuda, x, u, **kw)
    check(cuda, torch.full((9, 70000), 3.0), u, **kw)


def test_borders_of_two_tokens(cuda):
    """Weights 1 and 1/2 exactly (a logit difference of log 2 in fp64 is not exact: equal logits and none)."""
    x = torch.tensor([[0., 0., -math.inf, 0., 0.]])
    for v, want in ((0.0, 0), (0.25, 1), (0.5, 3), (0.75, 4), (0.7499, 3), (0.2499, 0)):
        assert sample(x.to(cuda), torch.tensor([v], device=cuda)).tolist() == [want]


def test_rows_with_nothing_and_with_infinities(cuda):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, -inf, -inf, -inf], [nan, nan, -inf, nan], [nan, -inf, 2., -inf], [inf, 1., inf, 2.],
                      [-inf, -3e38, -inf, -inf], [inf, nan, inf, -inf], [3e38, -3e38, 3e38, 1.]])
    u = torch.full((7,), 0.75)
    for kw in (dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=3, top_p=0.9)):
        out = check(cuda, x, u, **kw)
        assert out[:2].tolist() == [-1, -1]
    big = torch.full((2, 60000), -inf)
    big[1, 59999] = -5.0
    for kw in (dict(), dict(top_k=10), dict(top_p=0.5), dict(temperature=0.0)):
        assert check(cuda, big, u[:2], **kw).tolist() == [-1, 59999]


def test_random_numbers_at_and_past_their_ends(cuda):
    x, _ = rows_of(4, 3000, torch.float32, 6)
    u = torch.tensor([0.0, 1.0, -0.5, 7.0])
    out = sample(x.to(cuda), u.to(cuda), top_k=10).tolist()
    want = [drawn(r, v, 1.0, 10, 1.0, 0.0) for r, v in zip(x, (0.0, 1.0, 0.0, 1.0))]
    assert out == want
    fine = torch.rand(4, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    check(cuda, x, fine, top_p=0.97)


def test_parameters_per_row(cuda):
    x, u = rows_of(6, 2000, torch.bfloat16, 7)
    t = torch.tensor([0.5, 1.0, 0.0, 2.0, 0.8, 1.5])
    k = torch.tensor([0, 5, 3, 2000, 1, 40], dtype=torch.int32)
    p = torch.tensor([0.9, 1.0, 0.5, 0.25, 0.9, 0.75])
    m = torch.tensor([0.0, 0.125, 0.0, 0.0, 0.0, 0.03125])
    out = sample(x.to(cuda), u.to(cuda), t.to(cuda), k.to(cuda), p.to(cuda), m.to(cuda)).tolist()
    assert out == [drawn(x[i], u[i].double().item(), t[i].item(), int(k[i]), p[i].item(), m[i].item()) for i in range(6)]


def test_strides_offsets_and_shapes(cuda):
    x, u = rows_of(12, 1001, torch.bfloat16, 8)
    base = torch.zeros(12, 1300, dtype=torch.bfloat16)
    for start in (0, 1, 2, 3, 7):
        base[:, start:start + 1001] = x
        dev = base.to(cuda)[:, start:start + 1001]
        want = [drawn(r, v, 1.0, 0, 0.9, 0.0) for r, v in zip(x, u.double().tolist())]
        assert sample(dev, u.to(cuda), top_p=0.9).tolist() == want
    cube = sample(x.view(3, 4, 1001).to(cuda), u.view(3, 4).to(cuda), top_p=0.9)
    assert cube.shape == (3, 4) and cube.flatten().tolist() == want
    column = x.t().contiguous().to(cuda).t()  # the vocabulary is not the inner axis in memory
    assert sample(column, u.to(cuda), top_p=0.9).tolist() == want
    one = sample(x[0].to(cuda), u[0].to(cuda), top_p=0.9)
    assert one.shape == () and one.item() == want[0]
    assert sample(x[:0].to(cuda), u[:0].to(cuda)).shape == (0,)
    same = x[:1].to(cuda).expand(12, 1001)  # rows with a stride of zero
    assert sample(same, u.to(cuda)).tolist() == [drawn(x[0], v, 1.0, 0, 1.0, 0.0) for v in u.double().tolist()]


def test_frequencies(cuda):
    """Drawn with 2^16 evenly spaced numbers, every kept token comes as often as its weight says, to one draw."""
    x, _ = rows_of(1, 50, torch.float32, 9, spread=1.0)
    n = 1 << 16
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    out = sample(x.to(cuda).expand(n, 50), u.to(cuda), temperature=0.7, top_k=20)
    w = torch.softmax(x[0].double() / 0.7, 0)
    keep = x[0].argsort(descending=True)[:20]
    want = torch.zeros(50, dtype=torch.float64)
    want[keep] = w[keep] / w[keep].sum() * n
    assert ((torch.bincount(out.cpu(), minlength=50) - want).abs() <= 1.0).all()


def test_captured_and_replayed(cuda):
    x, u = (t.to(cuda) for t in rows_of(3, 5000, torch.bfloat16, 10))
    sample(x, u, top_k=50, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample(x, u, top_k=50, top_p=0.9)
        free = sample(x, u, top_p=0.9)
    for seed in range(4):
        nx, nu = rows_of(3, 5000, torch.bfloat16, 20 + seed)
        x.copy_(nx), u.copy_(nu)
        graph.replay()
        assert out.tolist() == sample(x, u, top_k=50, top_p=0.9).tolist()
        assert free.tolist() == sample(x, u, top_p=0.9).tolist()


def test_refusals(cuda):
    x, u = (t.to(cuda) for t in rows_of(3, 100, torch.float32, 11))
    for args, msg in [((x.half(), u), 'bfloat16'), ((x.cpu(), u), 'CUDA'), ((x, u[:2]), 'shape'), ((x, u.half()), 'float32'),
                      ((x, u.cpu()), 'beside'), ((x, u, -1.0), 'temperature'), ((x, u, float('nan')), 'temperature'),
                      ((x, u, 1.0, -1), 'top_k'), ((x, u, 1.0, 0, 0.0), 'top_p'), ((x, u, 1.0, 0, 1.5), 'top_p'),
                      ((x, u, 1.0, 0, 1.0, -0.1), 'min_p'), ((x, u, 1.0, 0, 1.0, 1.1), 'min_p'),
                      ((x, u, torch.ones(2, device=cuda)), 'temperature tensor'),
                      ((x, u, 1.0, torch.ones(3, device=cuda)), 'top_k tensor'), ((x[:, :0], u), 'vocab')]:
        with pytest.raises(ValueError, match=msg):
            sample(*args)


def test_temperatures_at_their_ends(cuda):
    """Exponents past every bin, weights that all round to the largest, and none at all."""
    x, u = rows_of(4, 3000, torch.float32, 12)
    for t in (1e-30, 1e-4, 1e-3, 0.01, 60.0, 1e4, 1e30, math.inf):
        for kw in (dict(), dict(top_k=9), dict(top_p=0.5), dict(top_k=1500, top_p=0.9, min_p=0.01)):
            check(cuda, x, u, temperature=t, **kw)
    check(cuda, x + 3e4, u, top_p=0.9)
    check(cuda, x - 3e4, u, top_p=0.9)
    check(cuda, x * 1e30, u, top_k=5)


def test_masked_stretches(cuda):
    """Most of the vocabulary at the type's lowest value, or at -infinity, as masks leave it."""
    for low, dtype in ((torch.finfo(torch.float32).min, torch.float32), (torch.finfo(torch.bfloat16).min, torch.bfloat16),
                       (-math.inf, torch.float32), (-1e9, torch.float32)):
        x, u = rows_of(3, 30000, torch.float32, 13)
        x[:, 300:29000] = low
        x[1, :29500] = low
        for kw in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(min_p=0.1)):
            check(cuda, x.to(dtype), u, **kw)


def test_more_equal_logits_at_a_cut_than_a_list_holds(cuda):
    x = torch.zeros(3, 40000)
    x[:, ::4], x[:, 1::4] = 1.0, 2.0
    u = torch.tensor([0.1, 0.5, 0.95])
    for kw in (dict(top_k=15000), dict(top_p=0.7), dict(top_k=25000, top_p=0.75), dict(min_p=0.3), dict(min_p=math.exp(-1) * 0.999)):
        check(cuda, x, u, **kw)
