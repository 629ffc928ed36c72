"""Paged attention held to what its weights keep, packed rows of inputs in all forms, and moves that are taken.

Bounds as in test_gpu_paged, with the weights' part by precision and output: 24 bits (three bf16 values, each rounded by at most 2^-8 of
what is left: 2^-24) where either is fp32; at precision and output bf16 16 bits (2^-16), or one bf16 value (2^-8) where a sequence, or
the branches over the pages that they share, has more than 160 query rows of a KV head.
"""
import math

import numpy as np
import pytest
import torch

from conftest import announce
from dkv import PagedCache, _lib
from test_gpu_paged import Model, rows_like

pytestmark = pytest.mark.gpu


def worst(m, step, q, k, v, out, many=()):
    """The largest error of `out` [tokens, q_heads, 64] in units of its bound; many: sequences whose weights are one bf16 value."""
    fp32, G, at, most = out.dtype == torch.float32, m.q_heads // m.heads, 0, 0.0
    for s, n in zip(step.seqs, step.counts):
        hist = m.k[s].shape[1] - n
        weights = 2 ** -24 if fp32 or m.precision == 'fp32' else 2 ** -8 if s in many or n * G > 160 else 2 ** -16
        for h in range(m.heads):
            keys, values = m.k[s][h, :hist], m.v[s][h, :hist]
            if m.precision == 'bf16':
                keys, values = keys.bfloat16(), values.bfloat16()
            keys, values = torch.cat((keys.double(), k[h, at:at + n].double())), torch.cat((values.double(), v[h, at:at + n].double()))
            x = q[h * G:(h + 1) * G, at:at + n].double()
            later = torch.arange(hist + n)[None] > hist + torch.arange(n)[:, None]
            p = torch.softmax((torch.matmul(x, keys.t()) / 8).masked_fill(later, -math.inf), -1)
            size = (torch.matmul(x.abs(), keys.abs().t()) / 8).masked_fill(later, 0).amax(-1, keepdim=True)
            e = 66 * 2 ** -24 * size + 2 ** -20 + weights
            ref = torch.matmul(p, values)
            tol = 2 * e * torch.matmul(p, values.abs()) + (2 ** -24 if fp32 else 2 ** -8) * ref.abs() + 1e-30
            got = out[at:at + n, h * G:(h + 1) * G].transpose(0, 1).double()
            most = max(most, ((got - ref).abs() / tol).nan_to_num(nan=math.inf).max().item())
        at += n
    return most


def attend(m, seqs, counts, out, many=()):
    step, k, v = m.step(seqs, counts, 16)
    q = (torch.randn(m.q_heads, step.tokens, 64, generator=m.gen) * 0.5).bfloat16()
    got = m.cache.attend(q[None].cuda(), k[None].cuda(), v[None].cuda(), 0, step, out_dtype=out)
    assert worst(m, step, q, k, v, got[0].cpu(), many) <= 1


KINDS = [('bf16', torch.bfloat16), ('bf16', torch.float32), ('fp32', torch.bfloat16), ('fp32', torch.float32)]


@pytest.mark.parametrize('precision,out', KINDS)
@pytest.mark.parametrize('counts', [1, [1, 2, 3, 4, 5, 1], [40, 1, 90, 64, 3, 33]])
def test_branches(cuda, counts, precision, out):
    """Few query rows over shared pages (15 to 45, 48 with the sequence apart) and many; the sequence apart is never of the group."""
    announce(f'branches {counts} {precision} {out}')
    m = Model(2, 6, precision)
    base = m.add()
    for bits, n in ((16, 40), (4, 300), (8, 333), (4, 64), (16, 30)):
        m.step(base, n, bits)
    seqs = [base] + m.cache.fork(base, 4)
    for s in seqs[1:]:
        m.k[s], m.v[s] = m.k[base], m.v[base]
    other = m.add()
    m.step([seqs[1], seqs[3], other], [3, 50, 100], 16)
    attend(m, seqs + [other], counts, out, many=seqs if counts == [40, 1, 90, 64, 3, 33] else ())
    attend(m, [seqs[2], other, seqs[0], seqs[4]], 1, out)


@pytest.mark.parametrize('precision,out', KINDS)
@pytest.mark.parametrize('branches', [53, 54, 100])
def test_single_tokens_of_many_branches(cuda, branches, precision, out):
    """159, 162 and 300 query rows over the pages in common: the last shapes of few rows, the first of many."""
    announce(f'{branches} branches {precision} {out}')
    m = Model(2, 6, precision, seed=branches, max_tokens=1 << 16)
    base = m.add()
    for bits, n in ((4, 500), (16, 70), (8, 700)):
        m.step(base, n, bits)
    seqs = m.cache.fork(base, branches)
    for s in seqs:
        m.k[s], m.v[s] = m.k[base], m.v[base]
    step = m.cache.step(seqs)
    assert (step.plan.long_work > 0) == (branches > 53)
    for s in seqs:  # (planned to look at it)
        m.cache.truncate(s, m.k[base].shape[1])
    attend(m, seqs, 1, out, many=seqs if branches > 53 else ())


@pytest.mark.parametrize('precision,out', KINDS)
def test_prompts_and_tokens_keep_their_weights(cuda, precision, out):
    announce(f'prompts and tokens {precision} {out}')
    m = Model(2, 6, precision, seed=8)
    seqs = [m.add() for _ in range(4)]
    m.step(seqs, [300, 64, 1, 700], [4, 8, 16, 4])
    for counts in ([53, 54, 1, 2], [1, 200, 53, 300], 1):
        attend(m, seqs, counts, out)


@pytest.mark.parametrize('bits', [4, 8, 16])
def test_rows_of_inputs_in_all_forms(cuda, bits):
    """Token-major rows, rows of a wider tensor, misaligned ones, fp32 and transposed ones: the same packed rows, read back."""
    announce(f'forms {bits}')
    heads, counts = 2, [1, 5, 100]
    gen = torch.Generator().manual_seed(bits)
    k, v = (rows_like(gen, 1, heads, sum(counts)).cuda() for _ in range(2))

    def wide(x, pad, at):
        y = torch.full((*x.shape[:3], 64 + pad), float('nan'), dtype=x.dtype, device='cuda')
        y[..., at:at + 64] = x
        return y[..., at:at + 64]
    forms = [lambda x: x, lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), lambda x: wide(x, 64, 8), lambda x: wide(x, 64, 3),
             lambda x: wide(x, 5, 2), lambda x: x.float(), lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)]
    m = Model(heads, heads)
    want = [m.stored(x[0].cpu(), bits) for x in (k, v)]
    for i, form in enumerate(forms):
        cache = PagedCache(1, heads, heads, max_tokens=4096)
        seqs = [cache.add() for _ in counts]
        cache.step(seqs, 7, bits)  # (not packed: the rows begin within a page)
        cache.append(form(k), form(v), 0, cache.step(seqs, counts, bits))
        got = cache.materialize(0, seqs, first=7, out_dtype=torch.float32)
        for x, y in zip(got, want):
            assert torch.equal(x[0].cpu(), y), i


MOVE = np.dtype([('src', '<i8'), ('dst', '<i8'), ('src_rows', 'u1'), ('src_row', 'u1'), ('dst_row', 'u1'), ('rows', 'u1'), ('bits', 'u1'),
                 ('reserved', 'u1', 3)])


@pytest.mark.parametrize('bits', [4, 8, 16])
@pytest.mark.parametrize('inside', [True, False])
def test_moves_that_are_taken(cuda, bits, inside):
    """Rows between pages of one arena and from tiles of another size elsewhere: two moves into neighbouring rows of a page, one tile read by
    two moves, rows moved within disjoint pages. Every byte that no move writes stays."""
    announce(f'moves {bits} inside={inside}')
    lib, layers, heads = _lib.load(), 2, 3
    subs, row = 2 * layers * heads, 8 * bits
    page = _lib.slab_bytes(64, bits, layers, heads)
    src_rows = 64 if inside else 33
    tile = _lib.slab_bytes(src_rows, bits, layers, heads)
    gen = torch.Generator().manual_seed(bits)
    dst = torch.randint(0, 256, (8 * page,), dtype=torch.uint8, generator=gen).cuda()
    src = dst if inside else torch.randint(0, 256, (3 * tile,), dtype=torch.uint8, generator=gen).cuda()
    first = 4 * page if inside else 0
    moves = [(first, 0, 5, 11, 17), (first, 0, 0, 28, 3), (first + tile, page, 32, 63, 1), (first + tile, 2 * page, 0, 0, 33),
             (first + 2 * tile, page, 1, 0, 31)]  # from, to, its row, to row, rows
    before, want = src.cpu().clone(), dst.cpu().clone()
    for a, b, r, to, n in moves:
        x, y = before[a:a + tile].view(subs, -1), want[b:b + page].view(subs, -1)
        y[:, to * row:(to + n) * row] = x[:, r * row:(r + n) * row]
        if bits < 16:
            y[:, 64 * row + 8 * to:64 * row + 8 * (to + n)] = x[:, src_rows * row + 8 * r:src_rows * row + 8 * (r + n)]
    m = np.array([(a, b, src_rows, r, to, n, bits, (0, 0, 0)) for a, b, r, to, n in moves], dtype=MOVE)
    _lib.check(lib.dkv_paged_move(src.data_ptr(), src.numel(), dst.data_ptr(), dst.numel(), m.ctypes.data, len(m), layers, heads,
                                  _lib.raw_stream(0)), 'dkv_paged_move')
    assert torch.equal(dst.cpu(), want)
