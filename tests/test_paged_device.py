"""generate_batch on a decoder whose device is not the current one, on the CPU: its forwards, captures and replays run with that device
current."""
import contextlib

import torch

from test_paged_streams import paged


class Device(str):
    """A place that tensors go to as to the CPU."""
    type = 'cuda'


def test_forwards_run_on_the_decoders_device(monkeypatch):
    current, seen = [], []

    @contextlib.contextmanager
    def device(x):
        current.append(x)
        yield
        current.pop()

    def forward(step, ids, last):
        seen.append(list(current))
        return torch.zeros(len(step.seqs), 10)
    d, pages, seq, _ = paged(monkeypatch, [[5, 6]] * 3, forward)
    monkeypatch.setattr(type(d), 'device', property(lambda self: Device('cpu')))
    monkeypatch.setattr(torch.cuda, 'device', device)
    d.generate_batch(pages, seq, [torch.tensor([[1, 2, 3]]), torch.tensor([[4]])], torch.zeros(2, 3))
    assert seen == [['cpu']] * 3 and not current
