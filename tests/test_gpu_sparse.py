"""attend_sparse and its index against the definitions in 64 bits: tile bounds bit for bit, the tiles each
query chooses, and attention over them, at ragged tiles, mixed widths, many or few query heads, chunk
segments, no index, an index older than the history, strided inputs and in graph replays."""
import pytest
import torch

from conftest import announce
from dkv.gpu_cache import GPUCache
from dkv.workloads import outlier_values
from oracle.attention import dequant_rows
from oracle.kv_quantization import pack_rows

pytestmark = pytest.mark.gpu

# (tokens, bits) of each append: a prefix, ragged frames, single tokens
RAGGED = [(39, 16), (64, 4), (78, 8), (1, 4), (130, 16), (64, 8), (17, 4), (63, 8), (200, 4), (64, 16)]


def build(cuda, segments, heads, layers=1, seed=0, precision='bf16', extra=256, gain=None):
    """A cache holding `segments`, and the dequantized history k, v [layers, heads, tokens, 64] fp32."""
    g = torch.Generator().manual_seed(seed)
    n = sum(s[0] for s in segments)
    k = outlier_values((layers * heads, n, 64), g, 0).view(layers, heads, n, 64)
    v = outlier_values((layers * heads, n, 64), g, 0).view(layers, heads, n, 64)
    c = GPUCache(None, layers=layers, heads=heads, max_tokens=n + extra, precision=precision)
    if n:
        c.append_batch(k.to(cuda), v.to(cuda), [b for _, b in segments], [t for t, _ in segments])
    dk, dv = [], []
    at = 0
    for t, b in segments:
        dk.append(dequant_rows(*pack_rows(k[:, :, at:at + t], b), b))
        dv.append(dequant_rows(*pack_rows(v[:, :, at:at + t], b), b))
        at += t
    empty = torch.zeros(layers, heads, 0, 64)
    return c, torch.cat(dk or [empty], 2), torch.cat(dv or [empty], 2)


def tiles_of(segments):
    out, at = [], 0
    for t, _ in segments:
        out += [(at + i, min(64, t - i)) for i in range(0, t, 64)]
        at += t
    return out


def chunk_of(heads, q_heads, nq, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    return (outlier_values((q_heads, nq, 64), g, 0), outlier_values((heads, nq, 64), g, 0),
            outlier_values((heads, nq, 64), g, 0))


def bounds_of(dk, tiles):
    """[tiles, layers, heads, 64] smallest and largest bf16 keys."""
    k = dk.to(torch.bfloat16).float()
    return tuple(torch.stack([f(k[:, :, a:a + n]) for a, n in tiles]) for f in
                 (lambda x: x.amin(2), lambda x: x.amax(2)))


def choice(q, low, high, blocks):
    """[heads, nq, tiles] bool: the definition, a query and tile at a time in 64 bits."""
    heads, tiles = low.shape[1], low.shape[0]
    qd = q.double().view(heads, -1, q.shape[1], 64)
    score = torch.zeros(heads, q.shape[1], tiles, dtype=torch.float64)
    for t in range(tiles):
        lo, hi = low[t].double()[:, None, None], high[t].double()[:, None, None]
        score[:, :, t] = torch.maximum(qd * lo, qd * hi).sum((1, 3))
    order = score.float().sort(dim=-1, descending=True, stable=True).indices
    return torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order[..., :blocks], True)


def expected(q, k, v, past, chosen_tokens, segments=None):
    """fp64 attention [nq, q_heads, 64]; chosen_tokens [heads, nq, past] bool; k, v [heads, past + nq, 64]."""
    heads, nq = k.shape[0], q.shape[1]
    part = torch.zeros(nq, dtype=torch.long)
    for b in (segments or [0, nq])[1:-1]:
        part[b:] += 1
    chunk = (part[:, None] == part[None]).tril()
    mask = torch.cat((chosen_tokens, chunk.expand(heads, nq, nq)), 2)[:, None]
    s = q.double().view(heads, -1, nq, 64) @ k.double()[:, None].transpose(2, 3) / 8
    p = torch.softmax(s.masked_fill(~mask, float('-inf')), -1)
    return (p @ v.double()[:, None]).reshape(q.shape[0], nq, 64).transpose(0, 1)


def tokens_of(chosen, tiles, past):
    out = torch.ones(*chosen.shape[:2], past, dtype=torch.bool)
    for t, (a, n) in enumerate(tiles):
        out[:, :, a:a + n] = chosen[:, :, t:t + 1]
    return out


def tolerance(ref, v, out_dtype, precision):
    """Per-element bound. An output is a mean of values: what its terms are off adds up to at most that much
    of the largest |v| of its head. p carries two bf16 terms (2^-17), the scores' sums of 64 products 64 * 2^-24
    of up to 2^6 (largest |s| here, exp makes it relative): 2^-12 in all; at fp32 v is off 2^-17 more. Then
    the output's own rounding."""
    big = v.abs().amax().double()
    off = big * (2.0 ** -17 + 2.0 ** -12 + 2.0 ** -17)
    return off + ref.abs() * (2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24)


def check(cuda, segments, heads, q_heads, nq, blocks, precision='bf16', out_dtype=torch.float32, indexed=None, parts=None,
          layer=0, layers=1, seed=0, strided=False):
    announce(f'sparse segments={len(segments)} heads={heads}/{q_heads} nq={nq} blocks={blocks} {precision} {out_dtype} '
             f'indexed={indexed} parts={parts} layer={layer}/{layers}')
    indexed = len(segments) if indexed is None else indexed
    first, rest = segments[:indexed], segments[indexed:]
    c, dk, dv = build(cuda, segments, heads, layers, seed, precision)
    if indexed < len(segments):  # the same history, indexed before the rest came
        whole = c
        c, _, _ = build(cuda, [], heads, layers, seed, precision, extra=whole.capacity)
        n = sum(t for t, _ in first)
        k, v = dk.to(torch.bfloat16).to(cuda), dv.to(torch.bfloat16).to(cuda)
        # (16-bit rows hold these bf16 values exactly)
        first, rest = [(t, 16) for t, _ in first], [(t, 16) for t, _ in rest]
        if n:
            c.append_batch(k[:, :, :n], v[:, :, :n], [16] * len(first), [t for t, _ in first])
        c.index()
        c.append_batch(k[:, :, n:], v[:, :, n:], [16] * len(rest), [t for t, _ in rest])
        dk, dv = k.float().cpu(), v.float().cpu()
    else:
        c.index()
    tiles = tiles_of(first)
    assert c.n_indexed == len(tiles)
    low, high = bounds_of(dk, tiles) if tiles else (torch.zeros(0, layers, heads, 64),) * 2
    got = c.tile_bounds()
    assert torch.equal(got[0].cpu().float(), low) and torch.equal(got[1].cpu().float(), high)
    q, kn, vn = chunk_of(heads, q_heads, nq, seed)
    past = dk.shape[2]
    for l in range(layers):
        c.select(16)
        c.append(kn[None].to(cuda), vn[None].to(cuda), l)
    qc, kc, vc = (t[None].to(cuda) for t in (q, kn, vn))
    if strided:  # [1, n, H, 64] projections seen as [1, H, n, 64]
        qc, kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (qc, kc, vc))
    out = c.attend_sparse(qc, kc, vc, layer, past, blocks, out_dtype=out_dtype, segments=parts)[0]
    assert out.shape == (nq, q_heads, 64) and out.dtype == out_dtype
    rounded = (lambda x: x.to(torch.bfloat16).float()) if precision == 'bf16' else (lambda x: x)
    k = torch.cat((rounded(dk[layer]), kn.float()), 1)
    v = torch.cat((rounded(dv[layer]), vn.float()), 1)
    chosen = choice(q, low[:, layer], high[:, layer], blocks) if tiles else torch.zeros(heads, nq, 0, dtype=torch.bool)
    ref = expected(q, k, v, past, tokens_of(chosen, tiles, past), parts)
    err = (out.cpu().double() - ref).abs()
    assert (err <= tolerance(ref, v, out_dtype, precision)).all(), err.max()
    return c, out


@pytest.mark.parametrize('precision', ['bf16', 'fp32'])
@pytest.mark.parametrize('blocks', [0, 1, 5, 100])
def test_single_token(cuda, precision, blocks):
    check(cuda, RAGGED, 5, 15, 1, blocks, precision)


@pytest.mark.parametrize('heads,q_heads', [(1, 1), (3, 9), (2, 14), (1, 16), (2, 34), (1, 40)])
def test_query_heads(cuda, heads, q_heads):
    check(cuda, RAGGED, heads, q_heads, 3, 4, 'bf16')


@pytest.mark.parametrize('precision', ['bf16', 'fp32'])
@pytest.mark.parametrize('nq', [2, 17, 64, 130])
def test_chunks(cuda, nq, precision):
    check(cuda, RAGGED, 5, 15, nq, 6, precision, torch.bfloat16 if nq == 64 else torch.float32)


def test_more_queries_than_split_workgroups(cuda):
    check(cuda, RAGGED, 8, 16, 193, 3, 'bf16')


@pytest.mark.parametrize('parts', [[0, 1, 70], [0, 30, 64, 69, 70]])
def test_chunk_segments(cuda, parts):
    check(cuda, RAGGED, 2, 6, 70, 4, 'fp32', parts=parts)


@pytest.mark.parametrize('segments', [[], [(1, 4)], [(64, 8)], [(65, 16)]])
def test_small_histories(cuda, segments):
    check(cuda, segments, 2, 6, 5, 2, 'fp32')


@pytest.mark.parametrize('indexed', [0, 4, 7])
def test_history_after_the_index(cuda, indexed):
    check(cuda, RAGGED + [(1, 16)] * 20, 3, 9, 4, 2, 'bf16', indexed=indexed)


@pytest.mark.parametrize('tail', [1, 63, 64, 65, 130])
def test_generated_tokens_after_the_index(cuda, tail):
    """Runs of one-row tiles, which are taken 64 at a time, with a frame among them or none."""
    check(cuda, RAGGED + [(1, 16)] * tail, 2, 6, 2, 3, 'fp32', indexed=10)
    check(cuda, RAGGED + [(1, 16)] * 5 + [(64, 16)] + [(1, 16)] * tail, 3, 9, 1, 2, 'bf16', indexed=10, layers=2, layer=1)
    check(cuda, [(65, 16)] + [(1, 16)] * tail, 1, 3, 3, 1, 'bf16', indexed=1)


def test_generated_tokens_at_other_widths_and_in_branches(cuda):
    """Only 16-bit rows lie evenly; a branch counts its own tiles, a reset cache none."""
    c, dk, dv = build(cuda, RAGGED + [(1, 8)] * 3 + [(1, 16)] * 4, 2)
    q, kn, vn = chunk_of(2, 6, 1, 7)
    qc, kc, vc = (t[None].to(cuda) for t in (q, kn, vn))
    past = dk.shape[2]
    k = torch.cat((dk[0].to(torch.bfloat16).float(), kn.float()), 1)
    v = torch.cat((dv[0].to(torch.bfloat16).float(), vn.float()), 1)
    ref = expected(q, k, v, past, torch.ones(2, 1, past, dtype=torch.bool))
    for cache in (c, c.fork()):
        cache.select(16)
        cache.append(kc, vc, 0)
        out = cache.attend_sparse(qc, kc, vc, 0, past, 2, out_dtype=torch.float32)
        assert ((out[0].cpu().double() - ref).abs() <= tolerance(ref, v, torch.float32, 'bf16')).all()
        assert cache.tile_singles[-5:] == [1, 2, 3, 4, 5]
    c.reset()
    c.select(4)
    for _ in range(3):
        c.append(kc, vc, 0)
    assert c.tile_singles == [0, 0, 0] and c._single_rows(3) == 0


def test_layers_and_strides(cuda):
    check(cuda, RAGGED, 3, 9, 9, 3, 'bf16', layers=3, layer=2, strided=True)


def test_many_tiles(cuda):
    check(cuda, [(64, b) for b in (4, 8, 16)] * 47 + [(3, 4)] * 70, 2, 6, 2, 33, 'bf16')


def test_equal_scores_choose_the_first_tiles(cuda):
    """Every frame has the same keys: all scores are equal, and the output is that of the first tiles."""
    g = torch.Generator().manual_seed(3)
    k1, v = torch.randn(2, 64, 64, generator=g), torch.randn(2, 64 * 20, 64, generator=g)
    k = k1.repeat(1, 20, 1).to(torch.bfloat16)
    c = GPUCache(None, layers=1, heads=2, max_tokens=2048)
    c.append_batch(k[None].to(cuda), v[None].to(torch.bfloat16).to(cuda), [16] * 20, [64] * 20)
    c.index()
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(2, 6, 3, 0))
    c.append(kn, vn, 0)
    out = c.attend_sparse(q, kn, vn, 0, 1280, 7)
    first = torch.zeros(2, 3, 1280, dtype=torch.bool)
    first[:, :, :7 * 64] = True
    ref = expected(q[0].cpu(), torch.cat((k.float(), kn[0].float().cpu()), 1),
                   torch.cat((v.to(torch.bfloat16).float(), vn[0].float().cpu()), 1), 1280, first)
    assert ((out[0].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 8 * 2.0 ** -11).all()


def test_a_past_inside_the_history(cuda):
    """A call over a part of the history: tiles that start later do not count, one that is cut is cut."""
    c, dk, dv = build(cuda, RAGGED, 2)
    c.index()
    q, kn, vn = chunk_of(2, 6, 2, 4)
    past = 39 + 64 + 40  # inside the third segment's first tile
    tiles = [t for t in tiles_of(RAGGED) if t[0] < past]
    low, high = bounds_of(dk, tiles)
    out = c.attend_sparse(q[None].to(cuda), kn[None].to(cuda), vn[None].to(cuda), 0, past, 2, out_dtype=torch.float32)
    k = torch.cat((dk[0, :, :past].to(torch.bfloat16).float(), kn.float()), 1)
    v = torch.cat((dv[0, :, :past].to(torch.bfloat16).float(), vn.float()), 1)
    ref = expected(q, k, v, past, tokens_of(choice(q, low[:, 0], high[:, 0], 2), tiles, past + 64)[:, :, :past])
    assert ((out[0].cpu().double() - ref).abs() <= tolerance(ref, v, torch.float32, 'bf16')).all()


def test_masked_rows_that_are_not_finite_stay_out(cuda):
    """NaN and infinity in chunk rows that a query does not see leave its output as it was."""
    c, dk, dv = build(cuda, RAGGED, 2)
    c.index()
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(2, 6, 8, 5))
    clean = c.attend_sparse(q, kn, vn, 0, c.seen[0], 3)
    kn, vn = kn.clone(), vn.clone()
    kn[:, :, 5], vn[:, :, 5] = float('nan'), float('inf')
    kn[:, :, 6], vn[:, :, 6] = float('inf'), float('nan')
    out = c.attend_sparse(q, kn, vn, 0, c.seen[0], 3)
    assert torch.equal(out[:, :5], clean[:, :5]) and torch.isfinite(clean).all()


def test_index_grows_with_the_history_and_branches_keep_theirs(cuda):
    c, dk, _ = build(cuda, RAGGED, 3, layers=2, extra=64 * 200)
    assert c.index() == len(tiles_of(RAGGED))
    before = [t.clone() for t in c.tile_bounds()]
    branch = c.fork()
    g = torch.Generator().manual_seed(9)
    k = outlier_values((6, 64 * 130, 64), g, 0).view(2, 3, -1, 64).to(cuda)
    c.append_batch(k, k, [16] * 130, [64] * 130)
    n = c.n_indexed
    assert c.index() == n + 130  # a larger buffer: two blocks of tiles more
    low, high = c.tile_bounds()
    assert torch.equal(low[:n], before[0]) and torch.equal(high[:n], before[1])
    x = k.view(2, 3, 130, 64, 64)
    assert torch.equal(low[n:], x.amin(3).permute(2, 0, 1, 3)) and torch.equal(high[n:], x.amax(3).permute(2, 0, 1, 3))
    assert all(torch.equal(a, b) for a, b in zip(branch.tile_bounds(), before))
    c.index(first=0)
    assert all(torch.equal(a, b) for a, b in zip(c.tile_bounds(), (low, high)))
    c.reset()
    assert c.n_indexed == 0 and c.tile_bounds()[0].shape[0] == 0


def test_a_planned_tile_that_fills_up_is_not_indexed_yet(cuda):
    c = GPUCache([(16, 64), (16, 70)], layers=1, heads=2)
    k = torch.randn(1, 2, 134, 64, device=cuda, dtype=torch.bfloat16)
    for a, b, n in ((0, 64, 1), (64, 100, 1), (100, 128, 2), (128, 131, 2), (131, 134, 3)):
        c.append(k[:, :, a:b], k[:, :, a:b], 0)
        assert c.index() == n
    assert torch.equal(c.tile_bounds()[0][2, 0], k[0, :, 128:].amin(1))


def test_attend_takes_the_sparse_path_where_the_cache_asks(cuda):
    c, _, _ = build(cuda, RAGGED, 3)
    c.index()
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(3, 9, 4, 6))
    past = c.seen[0]
    want = c.attend_sparse(q, kn, vn, 0, past, 3)
    c.sparse_blocks = 3
    assert torch.equal(c.attend(q, kn, vn, 0, past), want)
    assert not torch.equal(c.attend(q, kn, vn, 0, past, path='mfma'), want)


def test_another_stream(cuda):
    c, out = check(cuda, RAGGED, 5, 15, 3, 4, 'bf16', torch.bfloat16)
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(5, 15, 3, 0))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [c.attend_sparse(q, kn, vn, 0, c.seen[0] - 3, 4) for _ in range(3)]
    here = c.attend_sparse(q, kn, vn, 0, c.seen[0] - 3, 4)
    torch.cuda.synchronize()
    assert all(torch.equal(a[0], out) for a in again + [here])


def test_replays_follow_the_history_and_the_index(cuda):
    """One captured single-token call, replayed as tokens come and the index is renewed, gives what eager
    calls give, with eager work in between."""
    c, _, _ = build(cuda, RAGGED, 3, extra=400)
    c.index()
    g = torch.Generator().manual_seed(11)
    steps = [tuple(outlier_values((h, 1, 64), g, 0)[None].to(cuda) for h in (9, 3, 3)) for _ in range(9)]
    q, kn, vn = (t.clone() for t in steps[0])
    graph_steps = c.begin_graph_steps(1, q_heads=9)
    past = c.graph_step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.append(kn, vn, 0)
        out = c.attend_sparse(q, kn, vn, 0, past, 3)
    graph_steps.upload()
    graph.replay()
    c.end_graph_steps()
    for i, (qi, ki, vi) in enumerate(steps):
        if i:
            c.begin_graph_steps(1, steps=graph_steps)
            past = c.graph_step()
            for a, b in ((q, qi), (kn, ki), (vn, vi)):
                a.copy_(b)
            graph.replay()
            c.end_graph_steps()
        eager = c.attend_sparse(qi, ki, vi, 0, past, 3)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        if i == 4:
            n = c.n_indexed
            assert c.index() == n + 5


def test_replays_refuse_another_index(cuda):
    c, _, _ = build(cuda, RAGGED, 3, extra=64 * 300)
    c.index()
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(3, 9, 1, 0))
    c.begin_graph_steps(1, q_heads=9)
    past = c.graph_step()
    c.append(kn, vn, 0)
    c.attend_sparse(q, kn, vn, 0, past, 3)
    with pytest.raises(ValueError, match='graph steps'):
        c.index()
    steps = c.end_graph_steps()
    k = torch.randn(1, 3, 64 * 200, 64, device=cuda, dtype=torch.bfloat16)
    c.append_batch(k, k, [4] * 200, [64] * 200)
    c.index()
    c.begin_graph_steps(1, steps=steps)
    with pytest.raises(ValueError, match='capture again'):
        c.graph_step()


def test_refusals(cuda):
    c, _, _ = build(cuda, RAGGED, 3)
    q, kn, vn = (t[None].to(cuda) for t in chunk_of(3, 9, 4, 6))
    past = c.seen[0]
    for args, msg in [((q, kn, vn, 0, past, -1), 'blocks'), ((q[:, :8], kn, vn, 0, past, 1), 'multiple'),
                      ((q, kn[:, :2], vn, 0, past, 1), 'shape'), ((q, kn, vn[:, :, :3], 0, past, 1), 'shape'),
                      ((q, kn, vn, 1, past, 1), 'layer'), ((q, kn, vn, 0, past + 1, 1), 'longer'),
                      ((q, kn, vn, 0, -1, 1), 'longer'), ((q.cpu(), kn, vn, 0, past, 1), 'CUDA')]:
        with pytest.raises(ValueError, match=msg):
            c.attend_sparse(*args)
    with pytest.raises(ValueError, match='dtype'):
        c.attend_sparse(q, kn, vn, 0, past, 1, out_dtype=torch.float16)
    with pytest.raises(ValueError, match='segments'):
        c.attend_sparse(q, kn, vn, 0, past, 1, segments=[0, 3])
    with pytest.raises(ValueError, match='first'):
        c.index(first=c.n_indexed + 1)
    assert c.attend_sparse(q[:, :, :0], kn[:, :, :0], vn[:, :, :0], 0, past, 1).shape == (1, 0, 9, 64)
