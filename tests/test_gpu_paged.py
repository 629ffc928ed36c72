"""PagedCache on the GPU: packing, attention of many sequences over pages, adopting, forking, compacting, freeing.

Rows are compared with the oracle quantizer's, attention with softmax in 64 bits over its dequantized rows. Bounds of
the attention: a query's weights are off by a relative e, its output by at most 2 e times the weighted sum of |v|
(numerator and denominator), and by its own rounding (bf16 2^-8, fp32 2^-24). e: the score's products are exact and
their sums of 64 terms, with the scaling, are off by at most 66 roundings of 2^-24 of sum |q k| / 8, which enters the
exponent; exp2 and the sums of weights and products add 2^-20 at the lengths here; weights are kept in 16 bits (bf16
output) or 24 (fp32): 2^-16 and 2^-24, or, where a KV head has more than 160 query rows (tokens times query heads of a
sequence, or of branches over the pages that they share) at precision and output bf16, in one bf16 value: 2^-8.
"""
import math

import pytest
import torch

from conftest import announce
from dkv import GPUCache, PagedCache
from oracle.attention import dequant_rows
from oracle.kv_quantization import pack_rows

pytestmark = pytest.mark.gpu


def rows_like(gen, *shape):
    """K or V rows [..., tokens, 64] bf16 with a few loud channels, on the CPU."""
    x = torch.randn(*shape, 64, generator=gen)
    x[..., [3, 17, 40, 41]] *= 8
    return x.to(torch.bfloat16)


class Model:
    """What a cache of one layer should hold: for each sequence its dequantized rows, fp32 [heads, tokens, 64]."""

    def __init__(self, heads, q_heads, precision='bf16', max_tokens=1 << 15, layers=1, seed=0):
        self.cache = PagedCache(layers, heads, q_heads, max_tokens=max_tokens, precision=precision)
        self.gen = torch.Generator().manual_seed(seed)
        self.heads, self.q_heads, self.precision = heads, q_heads, precision
        self.k, self.v = {}, {}

    def add(self):
        seq = self.cache.add()
        self.k[seq] = self.v[seq] = torch.zeros(self.heads, 0, 64)
        return seq

    def stored(self, x, bits):
        x = x.contiguous()
        return dequant_rows(*pack_rows(x, bits), bits).float() if bits < 16 else x.float()

    def step(self, seqs, counts, bits, k=None, v=None, run=True):
        """A step whose rows are packed. Returns (step, k, v)."""
        step = self.cache.step(seqs, counts, bits)
        counts, bits = step.counts, step.bits
        if k is None:
            k, v = rows_like(self.gen, self.heads, sum(counts)), rows_like(self.gen, self.heads, sum(counts))
        if run:
            self.cache.append(k[None].cuda(), v[None].cuda(), 0, step)
        at = 0
        for s, n, w in zip(step.seqs, counts, bits):
            self.k[s] = torch.cat((self.k[s], self.stored(k[:, at:at + n], w)), 1)
            self.v[s] = torch.cat((self.v[s], self.stored(v[:, at:at + n], w)), 1)
            at += n
        return step, k, v

    def check(self, step, q, k, v, out, long=()):
        """`out` [tokens, q_heads, 64] of the last step against softmax in 64 bits. `long`: branches that share pages
        and have many query rows together."""
        fp32 = out.dtype == torch.float32
        at, G = 0, self.q_heads // self.heads
        worst = 0.0
        one = self.precision == 'bf16' and not fp32  # many rows' weights: one bf16 value
        for i, (s, n) in enumerate(zip(step.seqs, step.counts)):
            hist = self.k[s].shape[1] - n
            for h in range(self.heads):
                keys, values = self.k[s][h, :hist], self.v[s][h, :hist]
                if self.precision == 'bf16':
                    keys, values = keys.bfloat16(), values.bfloat16()
                keys = torch.cat((keys.double(), k[h, at:at + n].double()))
                values = torch.cat((values.double(), v[h, at:at + n].double()))
                x = q[h * G:(h + 1) * G, at:at + n].double()
                scores = torch.matmul(x, keys.t()) / 8
                later = torch.arange(hist + n)[None] > hist + torch.arange(n)[:, None]
                p = torch.softmax(scores.masked_fill(later, -math.inf), -1)
                size = (torch.matmul(x.abs(), keys.abs().t()) / 8).masked_fill(later, 0).amax(-1, keepdim=True)
                e = 66 * 2 ** -24 * size + 2 ** -20 + (2 ** -24 if fp32 else 2 ** -8 if one and (n * G > 160 or s in long) else 2 ** -16)
                ref = torch.matmul(p, values)
                tol = 2 * e * torch.matmul(p, values.abs()) + (2 ** -24 if fp32 else 2 ** -8) * ref.abs() + 1e-30
                got = out[at:at + n, h * G:(h + 1) * G].transpose(0, 1).double()
                ratio = ((got - ref).abs() / tol).nan_to_num(nan=math.inf).max().item()
                worst = max(worst, ratio)
                assert ratio <= 1, f'sequence {i} ({hist} + {n}), head {h}: {ratio:.3f} of the bound'
            at += n
        return worst

    def attend(self, seqs, counts, bits=16, out=torch.bfloat16, long=()):
        step, k, v = self.step(seqs, counts, bits)
        q = (torch.randn(self.q_heads, step.tokens, 64, generator=self.gen) * 0.5).bfloat16()
        got = self.cache.attend(q[None].cuda(), k[None].cuda(), v[None].cuda(), 0, step, out_dtype=out)
        assert got.shape == (1, step.tokens, self.q_heads, 64) and got.dtype == out
        return self.check(step, q, k, v, got[0].cpu(), long)


@pytest.mark.parametrize('heads', [1, 3, 8])
@pytest.mark.parametrize('bits', [4, 8, 16])
def test_packed_rows_are_the_quantizers(cuda, heads, bits):
    m = Model(heads, heads)
    seqs = [m.add() for _ in range(6)]
    for counts in ([1, 2, 63, 64, 65, 200], [1, 1, 1, 1, 1, 1], [70, 5, 64, 1, 130, 8]):
        announce(f'pack {heads} heads {bits} bits {counts}')
        step, k, v = m.step(seqs, counts, bits)
        got = m.cache.materialize(0, step, out_dtype=torch.float32)
        for x, y, have in ((got[0], k, m.k), (got[1], v, m.v)):
            at = 0
            for s, n in zip(seqs, counts):
                assert torch.equal(x[0, :, at:at + n].cpu(), have[s][:, -n:])
                at += n
    for s in seqs:
        k, v = m.cache.materialize(0, s, out_dtype=torch.float32)
        assert torch.equal(k[0].cpu(), m.k[s]) and torch.equal(v[0].cpu(), m.v[s])


def test_packed_bytes_are_the_packs(cuda):
    """The page of a 64-token frame holds what dkv_pack writes for it, every layer's, in bf16 strides of any order."""
    layers, heads = 3, 5
    gen = torch.Generator().manual_seed(5)
    for bits in (4, 8, 16):
        k = rows_like(gen, layers, 64, heads).cuda().transpose(1, 2)  # token-major
        v = rows_like(gen, layers, heads, 64).cuda()
        one = GPUCache(None, layers=layers, heads=heads, max_tokens=64)
        cache = PagedCache(layers, heads, heads, max_tokens=64)
        seq = cache.add()
        step = cache.step(seq, 64, bits)
        one.select(bits)
        for layer in range(layers):
            one.append(k[layer][None], v[layer][None], layer)
            cache.append(k[layer][None], v[layer][None], layer, step)
        n = 64 * {4: 40, 8: 72, 16: 128}[bits] * layers * 2 * heads
        at = (cache.pages(seq)[0][0] >> 2) * cache._info().grain
        assert torch.equal(cache.arena[at:at + n], one.arena[:n])


@pytest.mark.parametrize('precision,out', [('bf16', torch.bfloat16), ('bf16', torch.float32), ('fp32', torch.bfloat16),
                                           ('fp32', torch.float32)])
@pytest.mark.parametrize('heads,group', [(1, 1), (5, 3), (2, 16), (1, 20), (3, 7)])
def test_single_tokens(cuda, heads, group, precision, out):
    m = Model(heads, heads * group, precision, seed=heads)
    seqs = [m.add() for _ in range(7)]
    lengths = [1, 15, 64, 65, 200, 700]  # the last sequence has no history
    for bits in (4, 16, 8):
        m.step(seqs[:6], [n + bits for n in lengths], bits)
    for counts in (1, [1, 3, 1, 2, 1, 1, 1]):
        announce(f'single tokens {heads} x {group} {precision} {out} {counts}')
        m.attend(seqs, counts, 16, out)


@pytest.mark.parametrize('precision,out', [('bf16', torch.bfloat16), ('fp32', torch.float32)])
@pytest.mark.parametrize('counts', [[5, 60, 33], [1, 64, 65, 17], [130, 7, 257], [500]])
def test_prompts(cuda, counts, precision, out):
    m = Model(2, 6, precision, seed=len(counts))
    seqs = [m.add() for _ in counts]
    announce(f'prompts {counts} {precision} without a history')
    m.attend(seqs, counts, 8, out)
    announce(f'prompts {counts} {precision} after one')
    m.attend(seqs, counts[::-1], 4, out)
    m.attend(seqs, 1, 16, out)


def test_long_history(cuda):
    """Splits over many workgroups, pages of every width, a part page between widths."""
    m = Model(2, 8, 'bf16', max_tokens=1 << 16)
    seqs = [m.add(), m.add()]
    for i in range(12):
        m.step(seqs, [1000 + i, 77 * i + 1], (4, 8, 16)[i % 3])
    announce('long history')
    m.attend(seqs, 1)
    m.attend(seqs, [2, 1], 16, torch.float32)


@pytest.mark.parametrize('counts', [1, [1, 2, 3, 4, 5, 1], [40, 1, 90, 64, 3, 33]])
def test_branches_attend_to_what_they_share(cuda, counts):
    m = Model(2, 6)
    base = m.add()
    for bits, n in ((16, 40), (4, 300), (8, 333), (4, 64), (16, 30)):
        m.step(base, n, bits)
    seqs = [base] + m.cache.fork(base, 4)
    for s in seqs[1:]:
        m.k[s], m.v[s] = m.k[base], m.v[base]
    other = m.add()
    m.step([seqs[1], seqs[3], other], [3, 50, 100], 16)  # branches differ from here
    announce(f'branches {counts}')
    m.attend(seqs + [other], counts, 16, long=seqs + [other])
    m.attend(seqs + [other], 1, 16)
    m.attend([seqs[2], other, seqs[0], seqs[4]], 1, 8)  # in another order


def test_later_tokens_do_not_reach_a_query(cuda):
    """NaN and infinities in K and V of a later token, and in rows of pages that a sequence does not hold."""
    for bad in (math.nan, math.inf, -math.inf):
        for count, at in ((3, 2), (40, 21), (300, 170)):
            m = Model(2, 6, seed=count)
            m.cache.arena.view(torch.bfloat16).fill_(math.nan)
            seqs = [m.add(), m.add()]
            m.step(seqs, [70, 5], 16)
            m.step(seqs, [70, 5], 8)
            step, k, v = m.step(seqs, [count, 1], 16, run=False)
            q = (torch.randn(6, step.tokens, 64, generator=m.gen) * 0.5).bfloat16()
            k2, v2 = k.clone(), v.clone()
            k2[:, at, 5], v2[:, at, 9] = bad, bad
            announce(f'{bad} at {at} of {count}')
            out = m.cache.attend(q[None].cuda(), k2[None].cuda(), v2[None].cuda(), 0, step).cpu()
            clean = m.cache.attend(q[None].cuda(), k[None].cuda(), v[None].cuda(), 0, step).cpu()
            m.check(step, q, k, v, clean[0])
            same = [i for i in range(step.tokens) if not at <= i < count]
            assert torch.equal(out[0, same], clean[0, same])
            assert not out[0, at:count, :, 9].isfinite().all()


def test_visible_infinite_values(cuda):
    """A value that is infinite where rows of one block see it and others do not: as the formula has it."""
    m = Model(1, 3)
    seq = m.add()
    step, k, v = m.step(seq, 5, 16, run=False)
    v[0, 2, 9], v[0, 3, 10], v[0, 1, 11], v[0, 3, 11] = math.inf, math.nan, math.inf, -math.inf
    q = (torch.randn(3, 5, 64, generator=m.gen) * 0.5).bfloat16()
    out = m.cache.attend(q[None].cuda(), k[None].cuda(), v[None].cuda(), 0, step)[0].cpu()
    for i in range(5):
        for d in (9, 10, 11):
            seen = v[0, :i + 1, d].double()
            want = seen[~seen.isfinite()].sum()
            for got in out[i, :, d].double():
                assert got.isfinite() if want == 0 else (got.isnan() if want.isnan() else got == want)


def test_adopted_history(cuda):
    """Frames of other sizes than a page, generated tokens of a tile each, and a part of an evicted cache."""
    gen = torch.Generator().manual_seed(3)
    layers, heads = 3, 2
    one = GPUCache(None, layers=layers, heads=heads, max_tokens=2048)
    lengths = [50, 78, 78, 64, 17, 130] + [1] * 70
    bits = [16, 4, 4, 8, 8, 4] + [16] * 70
    k, v = rows_like(gen, layers, heads, sum(lengths)).cuda(), rows_like(gen, layers, heads, sum(lengths)).cuda()
    one.append_batch(k, v, bits, lengths)
    cache = PagedCache(layers, heads, 4, max_tokens=4096)
    seq = cache.adopt(one)
    assert cache.length(seq) == cache.position(seq) == sum(lengths)
    # 50 | 78 + 78 at 4 bits in three pages | 64 + 17 in two | 130 in three | 70 in two
    assert [r for _, r, _ in cache.pages(seq)] == [50, 64, 64, 28, 64, 17, 64, 64, 2, 64, 6]
    for layer in range(layers):
        for a, b in zip(cache.materialize(layer, seq), one.materialize(layer)):
            assert torch.equal(a, b)
    every = cache.materialize(None, seq)
    assert every[0].shape == (layers, heads, sum(lengths), 64)
    assert torch.equal(every[1][2:3], cache.materialize(2, [seq])[1])
    q = torch.randn(1, 4, 1, 64, generator=gen).bfloat16().cuda()
    step = cache.step(seq)
    kn, vn = k[1:2, :, :1], v[1:2, :, :1]
    mine = cache.attend(q, kn, vn, 1, step, out_dtype=torch.float32)
    theirs = one.attend(q, kn, vn, 1, sum(lengths), out_dtype=torch.float32, precision='fp32')
    assert (mine - theirs).abs().max() < 2 ** -7 * v.abs().max()  # (fp32 here rounds no row to bf16)
    one.mass().copy_(torch.rand(layers, heads, sum(lengths)))
    small = one.evict(200, sinks=50, recent=70)
    seq = cache.adopt(small)
    assert cache.length(seq) == 200 and cache.position(seq) == sum(lengths)
    for a, b in zip(cache.materialize(None, seq), zip(*(small.materialize(l) for l in range(layers)))):
        assert torch.equal(a, torch.cat(b))
    assert cache.step(seq, 2).positions.tolist() == [sum(lengths), sum(lengths) + 1]


def test_fork_truncate_compact_free(cuda):
    """Random calls against a plain model: what every sequence holds stays what was appended to it."""
    import random
    rng = random.Random(7)
    m = Model(2, 2, max_tokens=64 * 90)
    seqs = [m.add()]
    moved = 0
    for turn in range(150):
        kind = rng.choice(['step', 'step', 'step', 'fork', 'free', 'truncate', 'compact'])
        announce(f'turn {turn} {kind}')
        try:
            if kind == 'step':
                some = rng.sample(seqs, rng.randint(1, len(seqs)))
                m.step(some, [rng.choice([1, 3, 64, 100]) for _ in some], [rng.choice([4, 8, 16]) for _ in some])
            elif kind == 'fork':
                s = rng.choice(seqs)
                for b in m.cache.fork(s, rng.randint(0, 3)):
                    m.k[b], m.v[b] = m.k[s], m.v[s]
                    seqs.append(b)
            elif kind == 'free' and len(seqs) > 2:
                gone = rng.sample(seqs, rng.randint(1, len(seqs) - 1))
                m.cache.free(gone)
                seqs = [s for s in seqs if s not in gone]
            elif kind == 'truncate':
                s = rng.choice(seqs)
                n = rng.randint(0, m.cache.length(s))
                m.cache.truncate(s, n)
                m.k[s], m.v[s] = m.k[s][:, :n], m.v[s][:, :n]
            elif kind == 'compact':
                moved += m.cache.compact()
                info = m.cache.accounting()
                assert all(info['blocks'][w] == -(-info['pages'][w] // n) for w, n in ((4, 9), (8, 5), (16, 3)))
        except ValueError as e:  # full: nothing has changed
            assert 'full' in str(e)
            m.cache.free(seqs[1:])
            seqs = seqs[:1]
        if turn % 5 == 4:
            k, v = m.cache.materialize(0, seqs, out_dtype=torch.float32)
            assert torch.equal(k[0].cpu(), torch.cat([m.k[s] for s in seqs], 1))
            assert torch.equal(v[0].cpu(), torch.cat([m.v[s] for s in seqs], 1))
    assert moved
    m.cache.free(seqs)
    assert m.cache.accounting()['page_bytes'] == 0
