"""A PagedStep as the past_key_values of a decoder that nothing patched, on the CPU: refused by name."""
import pytest
import torch

from test_paged import Quiet


def test_an_unpatched_decoder_is_refused():
    transformers = pytest.importorskip('transformers')
    config = transformers.LlamaConfig(hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=1,
                                      num_key_value_heads=1, head_dim=64, vocab_size=16)
    model = transformers.LlamaModel(config).eval()
    c = Quiet(1, 1, 1)
    seq = c.add()
    step = c.step(seq, 3)
    with pytest.raises(ValueError, match='install_packed_attention'):
        model(input_ids=torch.zeros(1, 3, dtype=torch.int64), past_key_values=step, position_ids=step.positions[None])


@pytest.mark.parametrize('name,args', [('update', (None, None, 0)), ('crop', (1,)), ('reorder_cache', (None,)),
                                       ('batch_repeat_interleave', (2,)), ('batch_select_indices', (None,)), ('reset', ())])
def test_calls_on_a_cache_of_its_own_are_refused(name, args):
    c = Quiet(1, 1, 1)
    seq = c.add()
    step = c.step(seq, 3)
    with pytest.raises(ValueError, match=f'PagedStep.*{name}|{name}.*PagedStep'):
        getattr(step, name)(*args)
    assert c.length(seq) == 3
