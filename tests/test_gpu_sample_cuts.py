"""sample where two filters cut the same bin of weights."""
import math

import pytest
import torch

from conftest import announce
from dkv import gpu_ops
from test_gpu_sample import check, drawn

pytestmark = pytest.mark.gpu


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
