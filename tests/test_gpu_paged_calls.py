"""PagedCache's calls on the GPU in other circumstances: captured and replayed steps, other streams, strides, types and threads,
arenas and histories past 32 bits. Attention's bounds are those of test_gpu_paged."""
import threading

import pytest
import torch

from conftest import announce
from dkv import GPUCache, PagedCache
from test_gpu_paged import Model, rows_like

pytestmark = pytest.mark.gpu


def history(cache, layers, heads, gen):
    """Four sequences of which two share 300 tokens, every layer packed."""
    base, other, empty = cache.add(), cache.add(), cache.add()
    for counts, bits in (([200, 64], [8, 4]), ([100, 33], [4, 16])):
        step = cache.step([base, other], counts, bits)
        for layer in range(layers):
            cache.append(rows_like(gen, 1, heads, sum(counts)).cuda(), rows_like(gen, 1, heads, sum(counts)).cuda(), layer, step)
    return [base, *cache.fork(base), other, empty]


@pytest.mark.parametrize('counts', [1, [1, 3, 2, 1], [70, 9, 1, 130]])
def test_replayed_steps_are_eager_ones(cuda, counts):
    """Ten steps captured once and replayed after advance(), beside a second captured step over the same cache, with eager work
    and waits between, against eager steps of an equal cache: the same bits."""
    announce(f'replays {counts}')
    layers, heads, q_heads = 2, 2, 6
    caches, seqs = [], []
    for _ in range(2):
        caches.append(PagedCache(layers, heads, q_heads, max_tokens=1 << 14))
        seqs.append(history(caches[-1], layers, heads, torch.Generator().manual_seed(3)))
    mine, theirs = caches
    gen = torch.Generator().manual_seed(4)
    late = [mine.add(), theirs.add()]
    step = mine.step(seqs[0], counts, [16, 8, 4, 16], reserve=3000)
    second = mine.step(late[0], 5, 8, reserve=100)
    n = step.tokens

    def inputs(n):
        return [rows_like(gen, 1, h, n).cuda() for h in (q_heads, heads, heads)]
    q, k, v = inputs(n)
    q2, k2, v2 = inputs(5)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0]):
        for layer in range(layers):
            mine.append(k, v, layer, step)
            outs[0].append(mine.attend(q, k, v, layer, step))
    with torch.cuda.graph(graphs[1]):
        for layer in range(layers):
            outs[1].append(mine.attend(q2, k2, v2, layer, second, out_dtype=torch.float32))
            mine.append(k2, v2, layer, second)
    for turn in range(10):
        if turn:
            step.advance()
            second.advance()
            for x, y in zip((q, k, v, q2, k2, v2), inputs(n) + inputs(5)):
                x.copy_(y)
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        own = theirs.step(seqs[1], counts, [16, 8, 4, 16])
        own2 = theirs.step(late[1], 5, 8)
        assert torch.equal(own.positions, step.positions) and torch.equal(own2.positions, second.positions)
        for layer in range(layers):
            want = theirs.attend(q, k, v, layer, own)
            want2 = theirs.attend(q2, k2, v2, layer, own2, out_dtype=torch.float32)
            theirs.append(k, v, layer, own)
            theirs.append(k2, v2, layer, own2)
            assert torch.equal(outs[0][layer], want) and torch.equal(outs[1][layer], want2), (turn, layer)
        if turn % 3 == 0:
            torch.cuda.synchronize()
            for layer in range(layers):
                for a, b in zip(mine.materialize(layer, seqs[0] + late[:1]), theirs.materialize(layer, seqs[1] + late[1:])):
                    assert torch.equal(a, b)


def test_nothing_of_the_host_is_captured(cuda):
    cache = PagedCache(1, 1, 1, max_tokens=1024)
    seq = cache.add()
    step = cache.step(seq, 4)
    x = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device='cuda')
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.append(x, x, 0, step)
        for call in (lambda: cache.step(seq), step.advance, lambda: cache.fork(seq), lambda: cache.free(seq), lambda: cache.compact(),
                     lambda: cache.truncate(seq, 0), lambda: cache.materialize(0, seq)):
            with pytest.raises(ValueError, match='captured'):
                call()
    graph.replay()
    assert cache.length(seq) == 4
    cache.truncate(seq, 2)
    with pytest.raises(ValueError, match='since this step was planned'):
        cache.append(x, x, 0, step)
    with pytest.raises(ValueError, match='since this step was planned'):
        cache.attend(x, x, x, 0, step)


def test_other_streams(cuda):
    """Steps whose launches run on a stream of their own, which waits for the one before and which the next one waits for."""
    announce('streams')
    m = Model(2, 6, seed=9)
    seqs = [m.add() for _ in range(3)]
    side = torch.cuda.Stream()
    for i in range(6):
        stream = side if i % 2 else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream() if i % 2 else side)
        with torch.cuda.stream(stream):
            m.attend(seqs, [1, 40, 120], (4, 8, 16)[i % 3])
    torch.cuda.current_stream().wait_stream(side)
    step, k, v = m.step(seqs, 1, 16)  # planned here, launched there
    q = (torch.randn(6, 3, 64, generator=m.gen) * 0.5).bfloat16()
    args = [x[None].cuda() for x in (q, k, v)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = m.cache.attend(*args, 0, step)
    side.synchronize()
    m.check(step, q, k, v, out[0].cpu())


def test_strides_alignment_and_types(cuda):
    """The same values as token-major rows, rows of a wider tensor, misaligned ones, fp32 and one row that all heads and tokens
    share: the same bits."""
    announce('strides')
    heads, q_heads, counts = 2, 6, [1, 5, 100]
    gen = torch.Generator().manual_seed(2)
    n = sum(counts)
    q, k, v = (rows_like(gen, 1, h, n).cuda() for h in (q_heads, heads, heads))

    def wide(x, pad, at):
        y = torch.full((*x.shape[:3], 64 + pad), float('nan'), dtype=x.dtype, device='cuda')
        y[..., at:at + 64] = x
        return y[..., at:at + 64]
    forms = [lambda x: x, lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), lambda x: wide(x, 64, 8), lambda x: wide(x, 64, 3),
             lambda x: wide(x, 5, 2), lambda x: x.float(), lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)]
    outs = []
    for form in forms:
        cache = PagedCache(1, heads, q_heads, max_tokens=4096)
        seqs = [cache.add() for _ in counts]
        first = cache.step(seqs, counts, [4, 8, 16])
        cache.append(form(k), form(v), 0, first)
        step = cache.step(seqs, counts, 16)
        out = cache.attend(form(q), form(k), form(v), 0, step, out_dtype=torch.bfloat16)
        outs.append((out, *cache.materialize(0, seqs, first=0, out_dtype=torch.float32)))
        cache.append(form(k), form(v), 0, step)
    for other in outs[1:]:
        assert torch.equal(other[0], outs[0][0])
    cache = PagedCache(1, heads, q_heads, max_tokens=4096)
    seqs = [cache.add() for _ in counts]
    one = rows_like(gen, 1, 1, 1).cuda()
    step = cache.step(seqs, counts, 8)
    cache.append(one.expand(1, heads, n, 64), one.expand(1, heads, n, 64), 0, step)
    same = one.expand(1, heads, n, 64).contiguous()
    out = cache.attend(one.expand(1, q_heads, n, 64), one.expand(1, heads, n, 64), same, 0, step)
    assert torch.equal(out, cache.attend(one.expand(1, q_heads, n, 64).contiguous(), same, same, 0, step))
    got = cache.materialize(0, step, out_dtype=torch.float32)[0]
    assert torch.equal(got, got[:, :1, :1].expand_as(got))


def test_offsets_past_32_bits(cuda):
    """An arena of 12 GiB: pages of 8 MiB whose last layer and head lie past 2^32 bytes from its start, read in short and long
    steps, from branches, and moved."""
    announce('12 GiB arena')
    layers, heads, q_heads = 64, 8, 16
    cache = PagedCache(layers, heads, q_heads, max_tokens=64 * 1440)
    assert cache.arena_bytes > 11 << 30
    m = Model(heads, q_heads, seed=4)
    low, seq, between = cache.add(), cache.add(), cache.add()
    cache.step(low, 64 * 900, 16)  # 7 GiB of pages in front
    m.cache = _Last(cache, layers - 1)
    m.k[seq] = m.v[seq] = torch.zeros(heads, 0, 64)
    for n, bits in ((3000, 16), (500, 4), (700, 8)):
        m.step([seq], [n], bits)
    for _ in range(6):  # pages that leave gaps
        m.step([seq], [64], 16)
        cache.step(between, 128, 16)
    assert min(p >> 2 for p, _, _ in cache.pages(seq)) * cache._info().grain > 7 << 30
    m.attend([seq], 1)
    m.attend([seq], 90)
    branch = cache.fork(seq)[0]
    m.k[branch], m.v[branch] = m.k[seq], m.v[seq]
    m.attend([seq, branch], [3, 120], long=[seq, branch])
    cache.free([low, between])
    assert cache.compact() > 0
    k, v = cache.materialize(layers - 1, [seq, branch], out_dtype=torch.float32)
    for i, have in enumerate((m.k, m.v)):
        assert torch.equal((k, v)[i][0].cpu(), torch.cat((have[seq], have[branch]), 1))
    m.attend([branch, seq], 1)


class _Last:
    """A cache whose layer 0 is another one's `layer`."""

    def __init__(self, cache, layer):
        self.cache, self.layer = cache, layer
        self.step = cache.step

    def append(self, k, v, _, step):
        self.cache.append(k, v, self.layer, step)

    def attend(self, q, k, v, _, step, **kw):
        return self.cache.attend(q, k, v, self.layer, step, **kw)


def test_threads_of_one_process(cuda):
    """Caches of two threads, each on a stream of its own: what each gives alone."""
    announce('threads')

    def work(seed, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            m = Model(2, 6, seed=seed)
            seqs = [m.add() for _ in range(3)]
            for i in range(15):
                out.append(m.attend(seqs, [1, 2 + i, 60], (4, 8, 16)[i % 3]))
            torch.cuda.current_stream().synchronize()
    results = [[], []]
    threads = [threading.Thread(target=work, args=(s, results[s])) for s in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert [len(r) for r in results] == [15, 15]


def test_tokens_behind_the_last_sequence_stay(cuda):
    """Outputs and pages beyond a step's tokens are left as they were."""
    announce('rows behind')
    cache = PagedCache(1, 1, 3, max_tokens=1024)
    seqs = [cache.add(), cache.add()]
    cache.arena.fill_(0xA5)
    step = cache.step(seqs, [70, 3], 8)
    x = torch.randn(1, 1, 73, 64, device='cuda').bfloat16()
    cache.append(x, x, 0, step)
    grain = cache._info().grain
    page, rows = cache.pages(seqs[0])[1][:2]
    at = (page >> 2) * grain
    assert rows == 6
    codes, scales = cache.arena[at:at + 4096].view(64, 64), cache.arena[at + 4096:at + 4608].view(64, 8)
    assert (codes[6:] == 0xA5).all() and (scales[6:] == 0xA5).all()
    held = {p >> 2 for s in seqs for p, _, _ in cache.pages(s)}
    for block in range(cache.arena_bytes // grain // 48):
        for slot in range(5):
            g = 48 * block + 9 * slot
            if g not in held:
                assert (cache.arena[g * grain:(g + 9) * grain] == 0xA5).all()


@pytest.mark.parametrize('heads,group,counts', [(1, 1, [1]), (5, 3, [1] * 9), (2, 4, [70, 1, 64, 200, 3])])
def test_joined_projections(cuda, heads, group, counts):
    """Split, RoPE and pack in one launch: the rows of rope_qkv() and the bytes of append(), also replayed."""
    from dkv.gpu_ops import rope_qkv
    gen = torch.Generator().manual_seed(len(counts))
    n, q_heads = sum(counts), heads * group
    qkv = torch.randn(1, n, (q_heads + 2 * heads) * 64 + 64, generator=gen).bfloat16().cuda()[..., 64:]
    qkv[0, 0, -64:] = 0.0  # a row of one value, with a zero of each sign
    qkv[0, 0, -1] = -0.0
    angle = torch.rand(1, n, 32, generator=gen).repeat(1, 1, 2) * 50
    cos, sin = angle.cos().bfloat16().cuda(), angle.sin().bfloat16().cuda()
    for bits in (4, 8, 16):
        announce(f'joined projection {heads} x {group} {counts} {bits}')
        a, b = (PagedCache(3, heads, q_heads, max_tokens=4096) for _ in range(2))
        steps = []
        for cache in (a, b):
            cache.arena.zero_()
            seqs = [cache.add() for _ in counts]
            cache.step(seqs, 10, bits)
            steps.append(cache.step(seqs, counts, bits))
        q, k, v = rope_qkv(qkv, cos, sin, q_heads, heads)
        a.append(k, v, 1, steps[0])
        got = steps[1].append_projection(qkv, cos, sin, q_heads, 1)
        assert got[3] == 0 and all(torch.equal(x, y) for x, y in zip((q, k, v), got))
        assert torch.equal(a.arena, b.arena)
        b.arena.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = steps[1].append_projection(qkv, cos, sin, q_heads, 1)
        for _ in range(2):
            b.arena.zero_()
            graph.replay()
            assert torch.equal(a.arena, b.arena) and all(torch.equal(x, y) for x, y in zip((q, k, v), got))
    step = steps[1]
    for args in ((qkv[:, :, :64], cos, sin, q_heads, 1), (qkv.float(), cos, sin, q_heads, 1), (qkv, cos[..., :32], sin, q_heads, 1),
                 (qkv.cpu(), cos, sin, q_heads, 1), (qkv, cos, sin, q_heads + 1, 1)):
        assert step.append_projection(*args) is None
    with pytest.raises(ValueError, match='layer 3 of 3'):
        step.append_projection(qkv, cos, sin, q_heads, 3)


@pytest.mark.parametrize('q_heads,counts', [(200, [1, 2]), (300, [1, 1, 3]), (161, [1]), (64, [3, 1, 2])])
def test_many_query_heads_of_one(cuda, q_heads, counts):
    """One KV head with more query heads than a block has rows: a token's rows go over several blocks."""
    announce(f'{q_heads} query heads {counts}')
    m = Model(1, q_heads, seed=q_heads)
    seqs = [m.add() for _ in counts]
    for bits, n in ((4, 100), (16, 30), (8, 70)):
        m.step(seqs, n, bits)
    m.attend(seqs, counts)
    m.attend(seqs, counts, 8, torch.float32)


def test_adopted_branches_and_plans(cuda):
    """A fork's history with the tokens after it, and a planned cache that is filled up to the middle of a tile."""
    announce('adopted branches and plans')
    gen = torch.Generator().manual_seed(6)
    layers, heads = 2, 3
    rows = [rows_like(gen, 1, heads, n).cuda() for n in (100, 30, 1, 1)]
    base = GPUCache(None, layers=layers, heads=heads, max_tokens=1024)
    plan = GPUCache([(4, 100), (8, 90), (16, 30)], layers=layers, heads=heads)
    for cache, some in ((base, rows[:1]), (plan, rows)):
        for i, x in enumerate(some):
            cache.select(8 if i else 4)
            for layer in range(layers):
                cache.append(x, x, layer)
    fork = base.fork()
    for x in rows[1:]:
        fork.select(8)
        for layer in range(layers):
            fork.append(x, x, layer)
    pages = PagedCache(layers, heads, heads, max_tokens=2048)
    for cache, n in ((base, 100), (fork, 132), (plan, 132)):
        seq = pages.adopt(cache)
        assert pages.length(seq) == n
        for layer in range(layers):
            for x, y in zip(pages.materialize(layer, seq), cache.materialize(layer)):
                assert torch.equal(x, y)


def test_nothing_to_read(cuda):
    pages = PagedCache(2, 1, 1, max_tokens=256)
    seq = pages.add()
    for layer, shape in ((0, (1, 1, 0, 64)), (None, (2, 1, 0, 64))):
        assert [x.shape for x in pages.materialize(layer, [seq])] == [shape] * 2
    assert pages.fork(seq, 0) == [] and pages.compact() == 0
    assert pages.adopt(GPUCache(None, layers=2, heads=1, max_tokens=64)) != seq
    pages.free([])
    step = pages.step(seq, 3)
    assert pages.materialize(0, seq, first=3)[0].shape == (1, 1, 0, 64) and step.positions.tolist() == [0, 1, 2]


@pytest.mark.parametrize('precision,out', [('bf16', torch.bfloat16), ('fp32', torch.float32), ('fp32', torch.bfloat16), ('bf16', torch.float32)])
def test_prompts_beside_long_histories(cuda, precision, out):
    """Single tokens of long and short histories beside prompts: at fp32 too many units for one launch, at bf16 not, and few of them at
    both."""
    announce(f'prompts beside long histories {precision} {out}')
    m = Model(2, 6, precision, max_tokens=1 << 17, seed=11)
    seqs = [m.add() for _ in range(6)]
    m.step(seqs[:3], [40000, 30000, 20000], [4, 8, 4])
    m.step(seqs[3:5], [70, 200], 16)
    m.attend(seqs, [1, 2, 1, 100, 3, 300], 16, out)
    m.attend(seqs[3:], [90, 1, 2], 4, out)


@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('counts', [[1, 3], [70, 1, 200]])
def test_values_far_from_their_rows_middle(cuda, counts, bits, out):
    """One loud element a row puts the others at its edge. At precision fp32 a row is its middle plus scale * code, so what is summed
    is up to R = 2 max |v| of each row beside its values: products p * scale are off by 2^-24, weights kept in 24 bits by 2^-24, and a
    lane adds the middles of 32 keys a unit, the products of 16 keys in 3 terms each, which is 12 sums a unit of 16 products (their
    own sum taken as exact to 2^-23): 32 + 2 * 12 roundings of 2^-24 a unit of 64 keys, and 16 for the joins."""
    announce(f'values far from the middle {counts} {bits} {out}')
    m = Model(1, 3, 'fp32', seed=bits)
    seqs = [m.add() for _ in counts]
    n = 400 * len(counts)
    k, v = rows_like(m.gen, 1, n), (torch.rand(1, n, 64, generator=m.gen) * 2 - 1).bfloat16()
    v[..., 5] = -30
    v[..., 7::8] = 0.01
    m.step(seqs, 400, bits, k, v)
    step, k, v = m.step(seqs, counts, 16)
    q = (torch.randn(3, step.tokens, 64, generator=m.gen) * 0.5).bfloat16()
    got = m.cache.attend(q[None].cuda(), k[None].cuda(), v[None].cuda(), 0, step, out_dtype=out)[0].cpu().double()
    at = 0
    for s, c in zip(seqs, counts):
        keys, values = m.k[s][0].double(), m.v[s][0].double()
        later = torch.arange(400 + c)[None] > 400 + torch.arange(c)[:, None]
        x = q[:, at:at + c].double()
        p = torch.softmax((torch.matmul(x, keys.t()) / 8).masked_fill(later, float('-inf')), -1)
        size = (torch.matmul(x.abs(), keys.abs().t()) / 8).masked_fill(later, 0).amax(-1, keepdim=True)
        units = -(-400 // 64) + -(-c // 64)
        e = 66 * 2 ** -24 * size + 2 ** -20 + 2 ** -24
        ref = torch.matmul(p, values)
        spread = torch.matmul(p, 2 * values.abs().amax(-1, keepdim=True))
        tol = 2 * e * torch.matmul(p, values.abs()) + (2 + 56 * units + 16) * 2 ** -24 * spread + (2 ** -24 if out == torch.float32 else 2 ** -8) * ref.abs()
        ratio = ((got[at:at + c].transpose(0, 1) - ref).abs() / tol).max().item()
        assert ratio <= 1, (s, ratio)
        at += c
