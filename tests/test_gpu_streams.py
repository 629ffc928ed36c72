"""Long streams through the decoder on the GPU: what test_decoder_streams.py checks of the host, with the kernels."""
import pytest
import torch

from conftest import announce
from dkv.streaming import StreamingDecoder, build_decoder
from test_gpu_generate import SAMPLING, inputs
from test_gpu_streaming import SMALL, frames_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('graphs', [False, True])
def test_logits_that_are_not_numbers(cuda, graphs):
    announce(f'generate from NaN logits, graphs={graphs}')
    model = build_decoder(**SMALL, seed=3)
    dec = StreamingDecoder(model, graphs=graphs)
    prefix, question, u = inputs(4)
    cache = dec.ingest(prefix, frames_for(model, 2, seed=5), [4, 8])
    norm = model.model.norm.weight  # (NaN logits; the embeddings stay)
    norm.data.fill_(float('nan'))
    assert dec.generate(cache, question, u.cuda(), **SAMPLING).tolist() == [-1] * 12
    norm.data.fill_(1.0)
    assert min(dec.generate(cache, question, u.cuda(), **SAMPLING).tolist()) >= 0
