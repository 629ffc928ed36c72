"""A PagedCache's calls in several threads, on the CPU: what a call looks up and its launch are one section."""
import threading

import pytest
import torch

from dkv import PagedCache, _lib
from test_paged_streams import paged


LOCAL = threading.local()


class Held(PagedCache):
    """Bookkeeping alone, by the launches of the base class."""

    def __init__(self, monkeypatch, **kw):
        super().__init__(1, 1, 1, device='cpu', **kw)
        monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
        monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
        monkeypatch.setattr(_lib, 'raw_stream', lambda device=None: 0)
        self._arena_ptr = None

    # a device while this thread launches, none while it makes tensors
    _index = property(lambda self: getattr(LOCAL, 'index', -1), lambda self, index: None)

    def _launch(self, *a, **kw):
        LOCAL.index = 0
        try:
            return super()._launch(*a, **kw)
        finally:
            LOCAL.index = -1


@pytest.mark.parametrize('call', [lambda c, s: c.free(s), lambda c, s: c.truncate(s, 1), lambda c, s: c.compact(), lambda c, s: c.fork(s),
                                  lambda c, s: c.step(s, 3)])
def test_a_launch_keeps_other_threads_from_the_pages(monkeypatch, call):
    c = Held(monkeypatch)
    seq, other = c.add(), c.add()
    c.step([seq, other], 5)
    inside, go, done, errors = threading.Event(), threading.Event(), threading.Event(), []

    def launch(stream):
        inside.set()
        go.wait(10)
        assert not done.is_set()
        return 0

    def run(f):
        try:
            f()
        except Exception as e:
            errors.append(e)
    first = threading.Thread(target=run, args=(lambda: c._launch('a launch', launch),))
    first.start()
    assert inside.wait(10)
    second = threading.Thread(target=run, args=(lambda: (call(c, other), done.set()),))
    second.start()
    assert not done.wait(.2)
    go.set()
    first.join(10)
    second.join(10)
    assert done.is_set() and not errors, errors


def test_a_step_is_looked_at_where_it_is_launched(monkeypatch):
    c = Held(monkeypatch)
    seq, other = c.add(), c.add()
    step, calls = c.step(seq, 5), []
    c._launch('a launch', lambda stream: calls.append(1) or 0, 0, step)
    c.free(other)
    with pytest.raises(ValueError, match='since this step was planned'):
        c._launch('a launch', lambda stream: calls.append(1) or 0, 0, step)
    assert calls == [1]


def test_a_forward_of_all_questions_is_one_section(monkeypatch):
    """Another thread frees a sequence of the cache while a forward runs: behind it."""
    freed, order = [], []

    def forward(step, ids, last):
        t = threading.Thread(target=lambda: (pages.free(others.pop()), order.append('freed')))
        t.start()
        freed.append(t)
        t.join(.1)
        order.append('forward')
        assert step.generation == pages._generation.value
        return torch.zeros(len(step.seqs), 10)
    d, pages, seq, _ = paged(monkeypatch, [[5], [6], [7]], forward)
    others = [pages.add() for _ in range(3)]
    d.generate_batch(pages, seq, [torch.tensor([[1, 2, 3]])], torch.zeros(1, 3))
    for t in freed:
        t.join(10)
    assert order[0] == 'forward' and sorted(order) == ['forward'] * 3 + ['freed'] * 3
