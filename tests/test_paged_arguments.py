"""What a PagedCache's calls take as numbers, on the CPU."""
import numpy as np
import pytest
import torch

from test_paged import Quiet, rows


@pytest.mark.parametrize('bad', [1.7, [1.7], [1, 2.0], ['1'], None, [None], '1', [1, [2]], torch.tensor([1.5]), torch.tensor(1.5), np.float32(2)])
def test_counts_widths_and_first_tokens_are_whole_numbers(bad):
    c = Quiet(1, 1, 1)
    seqs = [c.add(), c.add()] if not isinstance(bad, list) or len(bad) == 2 else [c.add()]
    for call, what in ((lambda: c.step(seqs, bad), 'count'), (lambda: c.step(seqs, 1, bad), 'width'),
                       (lambda: c.materialize(0, seqs, bad), 'first token')):
        with pytest.raises(ValueError, match=what):
            call()
    assert all(c.length(s) == 0 for s in seqs)


def test_whole_numbers_of_any_type():
    c = Quiet(1, 1, 1)
    seqs = [c.add(), c.add()]
    for counts, bits in ((np.int64(3), np.int32(8)), (np.array([3, 3]), np.array([8, 8])), ((3, 3), (8, 8)),
                                        (torch.tensor([3, 3]), torch.tensor([8, 8])), (torch.tensor(3), torch.tensor(8))):
        c.step(seqs, counts, bits)
    assert [rows(c, s) for s in seqs] == [[15], [15]]


def test_a_refusal_names_the_value():
    c = Quiet(1, 1, 1)
    seqs = [c.add(), c.add()]
    with pytest.raises(ValueError, match='-2147483649'):
        c.step(seqs, [5, -(1 << 31) - 1])
    with pytest.raises(ValueError, match='2147483648'):
        c.step(seqs, [1 << 31, 3])
    with pytest.raises(ValueError, match='2 for 1'):
        c.step(seqs[:1], [1, 2])


@pytest.mark.parametrize('call', [lambda c, s: c.truncate(s, 1.5), lambda c, s: c.fork(s, 1.5), lambda c, s: c.step(s, reserve=1.5),
                                  lambda c, s: c.truncate(s, None), lambda c, s: c.fork(s, '2'), lambda c, s: c.step(s, reserve='x')])
def test_other_numbers_are_whole_too(call):
    c = Quiet(1, 1, 1)
    s = c.add()
    c.step(s, 5)
    with pytest.raises(ValueError, match='whole'):
        call(c, s)
    assert c.length(s) == 5 and c.accounting()['sequences'] == 1
