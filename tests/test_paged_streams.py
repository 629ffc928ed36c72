"""The decoder's host side over a PagedCache on the CPU: what is refused, and that branches end with the call."""
import types

import pytest
import torch

from dkv import streaming
from test_decoder_streams import decoder
from test_paged import Quiet


def paged(monkeypatch, drawn, forward=None):
    """A decoder whose forwards give zeros and whose draws are given, and a PagedCache with a history of 100 tokens."""
    seen = []

    def run(step, ids, last):
        seen.append((step.seqs, list(step.counts), ids.tolist(), step.positions.tolist()))
        return torch.zeros(len(step.seqs), 10)
    d = decoder(_paged_forward=forward or run, model=types.SimpleNamespace(lm_head=types.SimpleNamespace(weight=torch.zeros(1))))
    draws = iter(drawn)
    monkeypatch.setattr(streaming, 'sample', lambda *a: torch.tensor(next(draws)))
    pages = Quiet(2, 1, 2)
    seq = pages.add()
    pages.step(seq, 100, 4)
    return d, pages, seq, seen


def test_tokens_of_all_questions(monkeypatch):
    d, pages, seq, seen = paged(monkeypatch, [[5, 6], [-1, 7], [3, 8]])
    before = pages.accounting()
    out = d.generate_batch(pages, seq, [torch.tensor([[1, 2, 3]]), torch.tensor([[4]])], torch.zeros(2, 3))
    assert out.tolist() == [[5, -1, -1], [6, 7, 8]] and out.dtype == torch.int64
    assert [x[1:] for x in seen] == [([3, 1], [[1, 2, 3, 4]], [100, 101, 102, 100]), ([1, 1], [[5, 6]], [103, 101]),
                                     ([1, 1], [[0, 7]], [104, 102])]
    assert len(set(map(tuple, (x[0] for x in seen)))) == 1 and seq not in seen[0][0]
    assert pages.accounting() == before and pages.length(seq) == 100


def test_refusals(monkeypatch):
    d, pages, seq, seen = paged(monkeypatch, [])
    q, u = torch.tensor([[1, 2]]), torch.zeros(2, 3)
    for seqs, questions, x in (([seq], [q, q], u), (seq, [q], u), (seq, [q, q], u[0]), (seq, [q, q[:, :0]], u), (seq, [q, q[0]], u),
                               ([seq, 77], [q, q], u), (seq, [q, torch.zeros(2, 2, dtype=torch.int64)], u)):
        before = pages.accounting()
        with pytest.raises(ValueError):
            d.generate_batch(pages, seqs, questions, x)
        assert pages.accounting() == before
    assert not seen
    assert d.generate_batch(pages, seq, [q, q], u[:, :0]).shape == (2, 0)
    assert d.generate_batch(pages, [], [], u[:0]).shape == (0, 3)


def test_branches_end_with_an_error(monkeypatch):
    def fails(step, ids, last):
        raise RuntimeError('out of memory')
    d, pages, seq, _ = paged(monkeypatch, [], fails)
    before = pages.accounting()
    with pytest.raises(RuntimeError, match='out of memory'):
        d.generate_batch(pages, [seq, seq], [torch.tensor([[1, 2]])] * 2, torch.zeros(2, 3))
    assert pages.accounting() == before
    with pytest.raises(ValueError, match='full'):
        d.generate_batch(pages, [seq, seq], [torch.zeros(1, 100000, dtype=torch.int64)] * 2, torch.zeros(2, 3))
    assert pages.accounting() == before
