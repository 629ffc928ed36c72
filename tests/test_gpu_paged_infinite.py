"""Infinite and NaN values that a query sees, in the rows of its history at 16 bits and among the new tokens: what the formula makes of
them. A weight is positive, so an element is infinite where all such values that it sees have one sign and NaN otherwise; every other
element has the bits that it has without them, as no product of one column reaches another."""
import math

import pytest
import torch

from conftest import announce
from test_gpu_paged import Model, rows_like

pytestmark = pytest.mark.gpu

KINDS = [('bf16', torch.bfloat16), ('bf16', torch.float32), ('fp32', torch.bfloat16), ('fp32', torch.float32)]


def spoil(v, places):
    """Column 9: infinity at every place; 10: NaN at the first; 11: infinities of both signs in turn; 12: -infinity at the last."""
    bad = v.clone()
    for i, at in enumerate(places):
        bad[:, at, 9] = math.inf
        bad[:, at, 11] = -math.inf if i % 2 else math.inf
    if places:
        bad[:, places[0], 10] = math.nan
        bad[:, places[-1], 12] = -math.inf
    return bad


def expect(seen, clean):
    """The element of values `seen` [keys, 64] (fp64) whose clean output is `clean` [..., 64]."""
    want = clean.double().clone()
    for d in range(64):
        x = seen[:, d][~seen[:, d].isfinite()]
        if len(x):
            want[..., d] = x.sum()
    return want


def same(got, want):
    return torch.equal(got.double().nan_to_num(nan=7e77), want.nan_to_num(nan=7e77))


@pytest.mark.parametrize('precision,out', KINDS)
@pytest.mark.parametrize('past,in_past,count,in_new', [
    (0, [], 1, [0]),                       # a token alone
    (100, [], 1, [0]),
    (100, [0, 31, 32, 70], 1, []),         # in pages
    (700, [3, 699], 1, [0]),               # split over workgroups
    (40, [], 5, [0, 2, 3]),
    (0, [], 40, [0, 31, 32, 39]),          # several blocks of 16 query rows
    (130, [64], 60, [1, 59]),              # from here on more than 160 query rows
    (0, [], 100, [2, 63, 64, 85, 86, 99]), # both sides of a unit and of a block of 256 query rows
    (90, [89], 300, [0, 63, 128, 171, 299]),
    (0, [], 700, [5, 640]),                # split
    (1500, [700, 1499], 200, [100, 101]),
])
def test_visible_infinite_values(cuda, past, in_past, count, in_new, precision, out):
    announce(f'infinite values {past} {in_past} {count} {in_new} {precision} {out}')
    gen = torch.Generator().manual_seed(past + count)
    kp, vp = rows_like(gen, 2, past), rows_like(gen, 2, past)
    k, v = rows_like(gen, 2, count), rows_like(gen, 2, count)
    q = (torch.randn(6, count, 64, generator=gen) * 0.5).bfloat16()
    outs = []
    for spoilt in (False, True):
        m = Model(2, 6, precision)
        seq, other = m.add(), m.add()
        if past:
            m.step([seq], past, 16, kp, spoil(vp, in_past) if spoilt else vp)
        vn = spoil(v, in_new) if spoilt else v
        step = m.cache.step([seq], count)
        outs.append(m.cache.attend(q[None].cuda(), k[None].cuda(), vn[None].cuda(), 0, step, out_dtype=out)[0].cpu())
    clean, got = outs
    assert clean.isfinite().all()
    for h in range(2):
        seen = torch.cat((spoil(vp, in_past)[h], spoil(v, in_new)[h])).double()
        for i in range(count):
            rows = slice(3 * h, 3 * h + 3)
            assert same(got[i, rows], expect(seen[:past + i + 1], clean[i, rows])), (h, i)


@pytest.mark.parametrize('precision,out', KINDS)
@pytest.mark.parametrize('branches', [5, 60])
def test_infinite_values_in_shared_pages(cuda, branches, precision, out):
    """Branches whose shared pages hold them (few query rows together, and many), and whose own new rows do."""
    announce(f'infinite values of {branches} branches {precision} {out}')
    gen = torch.Generator().manual_seed(branches)
    kp, vp = rows_like(gen, 1, 640), rows_like(gen, 1, 640)
    k, v = rows_like(gen, 1, branches), rows_like(gen, 1, branches)
    q = (torch.randn(3, branches, 64, generator=gen) * 0.5).bfloat16()
    own = [1, branches - 1]
    outs = []
    for spoilt in (False, True):
        m = Model(1, 3, precision)
        base = m.add()
        m.step([base], 640, 16, kp, spoil(vp, [64, 639]) if spoilt else vp)
        step = m.cache.step(m.cache.fork(base, branches))
        vn = v.clone()
        if spoilt:
            vn[0, own, 20] = math.inf
        outs.append(m.cache.attend(q[None].cuda(), k[None].cuda(), vn[None].cuda(), 0, step, out_dtype=out)[0].cpu())
    clean, got = outs
    for i in range(branches):
        seen = torch.cat((spoil(vp, [64, 639])[0], v[0, i:i + 1])).double()
        if i in own:
            seen[-1, 20] = math.inf
        assert same(got[i], expect(seen, clean[i])), i


@pytest.mark.parametrize('precision,out', KINDS)
@pytest.mark.parametrize('count,at', [(3, 1), (40, 21), (300, 170)])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
def test_infinite_keys(cuda, bad, count, at, precision, out):
    """One element of a new token's key: rows that see the token have the formula's NaN, or lose the token where its score is minus
    infinity; the others keep their bits."""
    announce(f'key {bad} at {at} of {count} {precision} {out}')
    gen = torch.Generator().manual_seed(count)
    k, v = rows_like(gen, 2, count), rows_like(gen, 2, count)
    q = (torch.randn(6, count, 64, generator=gen) * 0.5).bfloat16()
    outs = []
    for spoilt in (False, True):
        m = Model(2, 6, precision)
        seqs = [m.add(), m.add()]
        m.step(seqs, [70, 5], 8, rows_like(torch.Generator().manual_seed(1), 2, 75), rows_like(torch.Generator().manual_seed(2), 2, 75))
        kn = k.clone()
        if spoilt:
            kn[:, at, 5] = bad
        step = m.cache.step([seqs[0]], count)
        outs.append(m.cache.attend(q[None].cuda(), kn[None].cuda(), v[None].cuda(), 0, step, out_dtype=out)[0].cpu())
    clean, got = outs
    assert torch.equal(got[:at], clean[:at])
    for i in range(at, count):
        for h in range(6):
            score = q[h, i, 5].float() * bad  # (the other products are finite)
            assert got[i, h].isfinite().all() if score == -math.inf else got[i, h].isnan().all(), (i, h)


@pytest.mark.parametrize('precision,out', KINDS)
@pytest.mark.parametrize('count', [1, 100])
@pytest.mark.parametrize('bits', [4, 8])
def test_packed_rows_without_a_scale(cuda, bits, count, precision, out):
    """A row packed from an infinite value has an infinite scale, which makes NaN of its codes of zero: elements that are NaN in the
    packed row stay NaN where a new token's value is infinite too."""
    announce(f'packed rows without a scale {bits} {count} {precision} {out}')
    gen = torch.Generator().manual_seed(bits)
    m = Model(1, 3, precision)
    seq = m.add()
    k, v = rows_like(gen, 1, 100), rows_like(gen, 1, 100)
    v[0, 70, 9] = math.inf
    m.cache.append(k[None].cuda(), v[None].cuda(), 0, m.cache.step(seq, 100, bits))
    stored = m.cache.materialize(0, seq, out_dtype=torch.float32)[1][0, 0].cpu()
    nan = stored.isnan().any(0)
    assert nan.sum() >= 62 and nan[20]
    k, v = rows_like(gen, 1, count), rows_like(gen, 1, count)
    v[0, count // 2, 20] = math.inf
    q = (torch.randn(3, count, 64, generator=gen) * 0.5).bfloat16()
    got = m.cache.attend(q[None].cuda(), k[None].cuda(), v[None].cuda(), 0, m.cache.step(seq, count), out_dtype=out)[0].cpu()
    assert got[..., nan].isnan().all()
