"""The decoder's host side over long streams on the CPU: caches whose launches are left out and a model that is not run."""
import types

import pytest
import torch

from dkv import streaming
from dkv.streaming import StreamingDecoder


class Branch:
    sparse_blocks = 0


def decoder(**kw):
    d = object.__new__(StreamingDecoder)
    d.__dict__.update(dict(graphs=False, pipeline=1, group_splits=None, precision='bf16', _cache=None, _spare=None, _graphs={},
                           _group_graphs={}, _qa_graphs={}, _qa_seen=set()), **kw)
    return d


def test_no_token_is_looked_up_where_none_could_be_drawn(monkeypatch):
    """A row without a token that can be drawn gives -1: that is never an index into the embeddings, and the tokens
    after it are -1 too."""
    drawn, looked_up = iter([5, -1, 7, -1, 2]), []

    def forward(branch, ids, logits):
        looked_up.append(ids.clone())
        return torch.zeros(1, 1, 10)
    d = decoder(_fork_forward=forward)
    monkeypatch.setattr(streaming, 'sample', lambda *a: torch.tensor([next(drawn)]))
    cache = types.SimpleNamespace(fork=Branch)
    out = d.generate(cache, torch.tensor([[3, 4]]), torch.zeros(5))
    assert out.tolist() == [5, -1, -1, -1, -1] and out.dtype == torch.int64
    assert all((ids >= 0).all() for ids in looked_up) and looked_up[1].tolist() == [[5]]
