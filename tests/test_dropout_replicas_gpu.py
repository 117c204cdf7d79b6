"""Dropout masks of replicas: one state, sites 2^48 apart."""
import pytest
import torch

import residual_oracle as ro
from test_transformer_joins_gpu import model, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_module():
    from spiky_b200 import residual

    x = torch.randn(7, 60, device=DEV)
    for replica in (None, 0, 3, 2 ** 15 - 1):
        y = residual.CounterDropout(0.25, seed=11, device=DEV, replica=replica)(x)
        kept = ro.keeps(0.25, 11, (replica or 0) << 48, x.numel()).view(x.shape)
        assert torch.equal(y.cpu() != 0, kept)


@pytest.mark.parametrize("batch_norm", [False, True])
def test_model(batch_norm):
    """A model's dropouts begin at its replica's site, one after another."""
    from spiky_b200 import lut_transformer

    seen = []
    for replica in (None, 2):
        m = model(dropout=0.5, counter_dropout=True, use_batch_norm=batch_norm, dropout_replica=replica).train()
        seen.clear()
        if batch_norm:
            with pytest.MonkeyPatch.context() as patch:
                real = lut_transformer._counter_dropout
                patch.setattr(lut_transformer, "_counter_dropout", lambda x, p, state, site: (seen.append(site), real(x, p, state, site))[1])
                out = m(tokens())
        else:
            hooks = [b.register_forward_pre_hook(lambda join, args: seen.append(args[3])) for n, b in m.named_modules() if n.endswith("_join")]
            out = m(tokens())
            assert len(hooks) == m._n_dropouts
        assert seen == [((replica or 0) << 48) + k for k in range(m._n_dropouts)] and out.isfinite().all()
    with pytest.raises(ValueError):
        model(dropout=0.5, dropout_replica=1)
    with pytest.raises(ValueError):
        model(dropout=0.5, counter_dropout=True, dropout_replica=-1)
