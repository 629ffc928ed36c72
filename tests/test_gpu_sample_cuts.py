"""sample where two filters cut the same bin of weights, and where the target lies among the lightest tokens that a sum
still counts."""
import math

import pytest
import torch

from conftest import announce
from dkv import gpu_ops
from test_gpu_sample import check, drawn

pytestmark = pytest.mark.gpu

NEAR_ONE = 1 - 2.0 ** -53


def close_rows(rows, vocab, step, seed):
    """Rows whose logits fall by `step` from token to token, in an order of their own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((rows, vocab), -40.0)
    for r in range(rows):
        at = torch.randperm(vocab, generator=g)[:800]
        x[r, at] = -step * torch.arange(800)
    return x


# An octave of weight has 8 bins: with steps of 1e-4, 800 tokens lie in one bin. min_p lies half a step from any token.
U = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.999, 1 - 2.0 ** -24])
CUTS = [(300, 600), (600, 300), (300, 301), (301, 300), (257, 799), (799, 257), (500, 500)]


@pytest.mark.parametrize('top_p', [1.0, 0.7, 0.999])
@pytest.mark.parametrize('top_k,tokens', CUTS)
def test_rank_and_min_p_cut_one_bin(cuda, top_k, tokens, top_p):
    """min_p leaves `tokens`, the rank top_k: the fewer of them stay, also behind a top_p."""
    min_p = math.exp(-1e-4 * (tokens - .5))
    for vocab in (1000, 30011):
        check(cuda, close_rows(6, vocab, 1e-4, top_k), U, top_k=top_k, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize('top_p', [1.0, 0.7])
@pytest.mark.parametrize('step', [1e-5, 1e-3, 1e-2])
def test_rank_and_min_p_of_wider_and_closer_logits(cuda, step, top_p):
    """The same in one step of a bin, in neighbouring bins and octaves apart."""
    for top_k, tokens in CUTS:
        check(cuda, close_rows(6, 5003, step, tokens), U, top_k=top_k, top_p=top_p, min_p=math.exp(-step * (tokens - .5)))


def test_rank_and_min_p_per_row(cuda):
    """As tensors of one value a row, ranks of the listed kind among them."""
    announce('sample, cuts per row')
    k = torch.tensor([300, 600, 40, 0, 257, 799], dtype=torch.int32)
    tokens = torch.tensor([600, 300, 600, 300, 799, 257])
    p = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.75, 0.75])
    m = torch.exp(-1e-4 * (tokens - .5))
    x = close_rows(6, 3000, 1e-4, 5)
    for u in (0.5, 0.999, 1 - 2.0 ** -24):
        us = torch.full((6,), u)
        out = gpu_ops.sample(x.to(cuda), us.to(cuda), 1.0, k.to(cuda), p.to(cuda), m.to(cuda)).tolist()
        assert out == [drawn(x[i], us[i].double().item(), 1.0, int(k[i]), p[i].item(), m[i].item()) for i in range(6)]


class Marked:
    """torch, whose empty int64 tensors hold a mark, so that a result nobody wrote shows."""
    MARK = -7

    def __getattr__(self, name):
        return getattr(torch, name)

    @staticmethod
    def empty(*args, **kw):
        x = torch.empty(*args, **kw)
        return x.fill_(Marked.MARK) if kw.get('dtype') is torch.int64 else x


@pytest.mark.parametrize('vocab,shift', [(8192, 48), (49280, 46), (131071, 45)])
@pytest.mark.parametrize('below', [-0.0009, 0.0, 0.0009, -0.4])
def test_target_among_the_lightest_tokens(cuda, vocab, shift, below, monkeypatch):
    """One logit at the top, the last 2048 at the weight that one unit of the sums has or `below` it, and a random
    number so near to one that it lies in their weight: the token is one that may be drawn. A sum counts in units of
    2^-shift of twice the largest weight, a border may lie as many of them off as there are tokens and bins' sums
    (64 parts of 401); where they are not lighter than a unit or about it, it is the last of them."""
    announce(f'sample, lightest tokens: vocab={vocab} below={below}')
    monkeypatch.setattr(gpu_ops, 'torch', Marked())
    x = torch.full((1, vocab), -math.inf)
    x[0, 5] = 0.0
    x[0, -2048:] = (1 - shift + below) * math.log(2)
    for u in (1.0, NEAR_ONE, 1 - 2.0 ** -40):
        for kw in (dict(), dict(top_p=1 - 2.0 ** -50), dict(min_p=1e-30), dict(top_k=1000), dict(top_k=3000), dict(top_k=100)):
            out = gpu_ops.sample(x.to(cuda), torch.tensor([u], dtype=torch.float64, device=cuda), **kw).tolist()
            if out[0] == Marked.MARK:
                pytest.fail(f'no token written: u={u} {kw}')
            assert out[0] == 5 or out[0] >= vocab - 2048, (u, kw)
            if u == 1 and below >= 0 and not kw:
                assert out[0] == vocab - 1, (u, kw)


@pytest.mark.parametrize('vocab', [8192, 49280, 131071])
def test_one_is_the_last_token_that_counts(cuda, vocab):
    """u of one over tokens at every distance from the largest, in parts far apart: the last one with weight."""
    announce(f'sample, u = 1: vocab={vocab}')
    x = torch.full((1, vocab), -math.inf)
    x[0, 0] = 0.0
    for at, low in ((vocab - 1, -20.0), (vocab // 2, -25.0), (vocab - 3000, -28.0), (vocab - 7, 0.0)):
        y = x.clone()
        y[0, at] = low
        got = gpu_ops.sample(y.to(cuda), torch.ones(1, dtype=torch.float64, device=cuda)).tolist()
        assert got == [at]


@pytest.mark.parametrize('kw', [dict(), dict(top_p=0.9), dict(top_k=500, min_p=1e-4), dict(top_k=50, top_p=0.95)],
                         ids=lambda kw: '-'.join(kw) or 'none')
def test_batches_of_other_sizes(cuda, kw):
    """Rows cut into other parts by the size of their batch: the same tokens, as none of these random numbers is within
    the sums' rounding of a border."""
    announce(f'sample, batch sizes: {kw}')
    g = torch.Generator().manual_seed(21)
    x, u = (torch.randn(700, 20011, generator=g) * 2.5).to(cuda), torch.rand(700, generator=g).to(cuda)
    whole = gpu_ops.sample(x, u, **kw)
    for rows in (1, 3, 40, 300):
        assert torch.equal(gpu_ops.sample(x[:rows], u[:rows], **kw), whole[:rows])
