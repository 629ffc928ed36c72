"""attention_mass and observe against softmax column sums in 64 bits: ragged tiles, mixed widths, many query
heads, chunk segments, long chunks, masked rows, accumulation, branches and graph replays."""
import pytest
import torch

from conftest import announce
from dkv.gpu_cache import GPUCache
from test_gpu_sparse import RAGGED, build, chunk_of

pytestmark = pytest.mark.gpu


def expected(q, k, past, segments=None):
    """fp64 column sums [heads, past + nq]; q [q_heads, nq, 64], k [heads, past + nq, 64]."""
    heads, nq = k.shape[0], q.shape[1]
    part = torch.zeros(nq, dtype=torch.long)
    for b in (segments or [0, nq])[1:-1]:
        part[b:] += 1
    mask = torch.cat((torch.ones(nq, past, dtype=torch.bool), (part[:, None] == part[None]).tril()), 1)
    s = q.double().view(heads, -1, nq, 64) @ k.double()[:, None].transpose(2, 3) / 8
    return torch.softmax(s.masked_fill(~mask, float('-inf')), -1).sum((1, 2))


def keys(dk, kn, precision, layer=0):
    k = dk[layer].to(torch.bfloat16).float() if precision == 'bf16' else dk[layer]
    return torch.cat((k, kn.float()), 1)


def check_close(out, ref):
    """Every weight's relative error: its score's (products exact or 2^-24 each, sums of 64 products of scores up
    to 2^6: 64 * 2^-24 * 2^6, a bound on sums that add in any order) and its row sum's (as much again): 2^-11;
    a column's sum adds less than 2^-16 of that. Sums that underflow are below 2^-100."""
    err = (out.cpu().double() - ref).abs()
    assert (err <= 2.0 ** -11 * ref + 2.0 ** -100).all(), (err / ref.clamp(min=1e-30)).max()
    # and on average far less: the errors above are 2^-9 of that bound, of either sign
    assert err.norm() <= 2.0 ** -18 * ref.norm(), err.norm() / ref.norm()


def check(cuda, segments, heads, q_heads, nq, precision='bf16', parts=None, strided=False, layers=1, layer=0):
    announce(f'mass segments={len(segments)} heads={heads}/{q_heads} nq={nq} {precision} parts={parts}')
    c, dk, _ = build(cuda, segments, heads, layers, precision=precision, extra=nq + 8)
    q, kn, _ = chunk_of(heads, q_heads, nq, 0)
    past = dk.shape[2]
    qc, kc = q[None].to(cuda), kn[None].to(cuda)
    if strided:
        qc, kc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (qc, kc))
    out = c.attention_mass(qc, kc, layer, past, segments=parts)
    assert out.shape == (heads, past + nq) and out.dtype == torch.float32
    check_close(out, expected(q, keys(dk, kn, precision, layer), past, parts))
    again = c.attention_mass(qc, kc, layer, past, segments=parts)
    assert torch.equal(out, again)
    return c, out


@pytest.mark.parametrize('precision', ['bf16', 'fp32'])
@pytest.mark.parametrize('nq', [1, 3, 16, 64, 65, 200])
def test_chunks(cuda, nq, precision):
    check(cuda, RAGGED, 5, 15, nq, precision)


@pytest.mark.parametrize('heads,q_heads', [(1, 1), (2, 14), (1, 40), (8, 8)])
def test_query_heads(cuda, heads, q_heads):
    check(cuda, RAGGED, heads, q_heads, 5, 'fp32')


@pytest.mark.parametrize('parts', [[0, 1, 70], [0, 30, 64, 69, 70]])
def test_chunk_segments(cuda, parts):
    check(cuda, RAGGED, 2, 6, 70, parts=parts)


@pytest.mark.parametrize('segments', [[], [(1, 4)], [(64, 8)], [(65, 16)], [(1, 16)] * 130])
def test_small_histories(cuda, segments):
    check(cuda, segments, 2, 6, 5, 'fp32')


def test_layers_and_strides(cuda):
    check(cuda, RAGGED, 3, 9, 9, strided=True, layers=3, layer=2)


def test_many_units(cuda):
    check(cuda, [(64, b) for b in (4, 8, 16)] * 70, 2, 6, 2, 'bf16')


def test_long_chunk(cuda):
    check(cuda, [(100, 8)], 2, 6, 700, 'bf16')


def test_masked_keys_that_are_not_finite_count_nothing(cuda):
    """What chunk keys behind a segment hold does not reach the tokens before it."""
    c, dk, _ = build(cuda, RAGGED, 2)
    q, kn, _ = chunk_of(2, 6, 8, 5)
    past = dk.shape[2]
    bad = kn.clone()
    bad[:, 5:] = float('nan')
    bad[:, 6] = float('inf')
    out = c.attention_mass(q[None].to(cuda), bad[None].to(cuda), 0, past, segments=[0, 5, 8])
    one = expected(q[:, :5], keys(dk, kn[:, :5], 'bf16'), past)
    part = c.attention_mass(q[None, :, :5].to(cuda), kn[None, :, :5].to(cuda), 0, past)
    check_close(part, one)
    assert torch.isnan(out[:, past + 7]).all()  # a key that its own query sees
    assert torch.isfinite(out[:, past:past + 5]).all()


def test_observe_accumulates_per_layer(cuda):
    c, dk, _ = build(cuda, RAGGED, 3, layers=2)
    past = dk.shape[2]
    q, kn, _ = chunk_of(3, 9, 6, 1)
    qc, kc = q[None].to(cuda), kn[None].to(cuda)
    one = [c.attention_mass(qc, kc, l, past) for l in range(2)]
    for _ in range(2):
        c.observe(qc, kc, 0, past)
    c.observe(qc, kc, 1, past)
    for l in range(2):
        c.append(kc, kc, l)
    m = c.mass()
    assert m.shape == (2, 3, past + 6)
    assert torch.equal(m[0], one[0] + one[0]) and torch.equal(m[1], one[1])
    branch = c.fork()
    branch.observe(qc, kc, 1, past)
    assert torch.equal(branch.mass()[1], one[1] + one[1]) and torch.equal(c.mass()[1], one[1])
    c.reset()
    assert c._mass.abs().sum() == 0


def test_attend_observes_where_the_cache_asks(cuda):
    c, _, _ = build(cuda, RAGGED, 3)
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(3, 9, 4, 6))
    past = c.seen[0]
    want = c.attend(q, kn, vn, 0, past)
    c.observing = True
    assert torch.equal(c.attend(q, kn, vn, 0, past), want)
    assert torch.equal(c._mass[0, :, :past + 4], c.attention_mass(q, kn, 0, past))
    assert not c.fork().observing


def test_replays_observe_as_eager_calls(cuda):
    c, _, _ = build(cuda, RAGGED, 3, extra=400)
    want = torch.zeros(3, c.capacity, device=cuda)
    c.mass()
    g = torch.Generator().manual_seed(2)
    chunks = [(torch.randn(1, 9, 4, 64, generator=g).to(torch.bfloat16).to(cuda),
               torch.randn(1, 3, 4, 64, generator=g).to(torch.bfloat16).to(cuda)) for _ in range(6)]
    q, kn = (t.clone() for t in chunks[0])
    steps = c.begin_graph_steps(4, q_heads=9)
    past = c.graph_step()
    with pytest.raises(ValueError, match='graph steps'):
        c.attention_mass(q, kn, 0, past)
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
            c.begin_graph_steps(4, steps=steps)
            past = c.graph_step()
            q.copy_(qi), kn.copy_(ki)
            graph.replay()
            c.end_graph_steps()
        want[:, :past + 4] += c.attention_mass(qi, ki, 0, past)
        torch.cuda.synchronize()
        assert torch.equal(c._mass[0], want), i
    branch = c.fork()
    branch.mass()
    branch.begin_graph_steps(4, steps=steps)
    with pytest.raises(ValueError, match='capture again'):
        branch.graph_step()


def test_refusals(cuda):
    c, _, _ = build(cuda, RAGGED, 3)
    q, kn, _ = (t[None].to(cuda) for t in chunk_of(3, 9, 4, 6))
    past = c.seen[0]
    for call in (c.attention_mass, c.observe):
        for args, msg in [((q[:, :8], kn, 0, past), 'multiple'), ((q, kn[:, :2], 0, past), 'shape'), ((q, kn, 1, past), 'layer'),
                          ((q, kn, 0, past + 1), 'longer'), ((q, kn.cpu(), 0, past), 'CUDA')]:
            with pytest.raises(ValueError, match=msg):
                call(*args)
    assert c.attention_mass(q[:, :, :0], kn[:, :, :0], 0, past).abs().sum() == 0
