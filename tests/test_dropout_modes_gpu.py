"""Counter dropout follows the mode of each block, as torch's dropout does, not that of the model alone."""
import pytest
import torch

from test_transformer_joins_gpu import model, tokens

pytestmark = pytest.mark.gpu


def same_twice(m):
    torch.manual_seed(1)
    return torch.equal(m(tokens()), m(tokens()))


@pytest.mark.parametrize("opts", [dict(counter_dropout=False), dict(), dict(use_batch_norm=True), dict(norm="rms", gated=True), dict(no_ffn=True)])
def test_modes_of_blocks(opts):
    opts = dict(dict(dropout=0.5, counter_dropout=True), **opts)
    m = model(**opts).train()
    assert not same_twice(m)
    for block in m.layers:
        block.eval()
    assert same_twice(m)
    m.layers[1]["attention_dropout"].train()
    if "attention_join" in m.layers[1]:
        m.layers[1]["attention_join"].train()
    assert not same_twice(m)
    m.eval()
    assert same_twice(m)
    for block in m.layers:   # (dropout alone, as a Monte Carlo estimate has it)
        for name, part in block.items():
            if name.endswith(("_dropout", "_join")):
                part.train()
    assert not same_twice(m)


def test_probability_of_zero():
    for opts in (dict(), dict(use_batch_norm=True), dict(norm="rms")):
        m = model(dropout=0.0, counter_dropout=True, **opts).train()
        state = m.dropout_state.clone()
        assert m.take_dropout_state() is None
        m(tokens())
        assert torch.equal(state, m.dropout_state)
