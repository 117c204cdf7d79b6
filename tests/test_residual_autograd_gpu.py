"""Residual-stream operators under what torch does around a call - traces, recomputation, forward mode, second derivatives - on both routes."""
import pytest
import torch

from test_residual_calls_gpu import routes  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def operators(residual):
    """Each operator as a function of one tensor [rows, C]."""
    state = residual.dropout_state(1, DEV)
    return dict(norm=lambda v: residual.row_norm(v), join=lambda v: residual.residual_join(v, v),
                normed=lambda v: residual.residual_join(v, v, branch_norm="layer", next_norm="rms")[1],
                dropout=lambda v: residual.counter_dropout(v, 0.5, state))


# ------------------------------------------------------------------------------------------------ recording
def test_traces_are_refused(routes):  # noqa: F811
    """What is recorded would lack the kernels: it would return memory that nobody wrote."""
    from spiky_b200 import residual
    from torch.fx.experimental.proxy_tensor import make_fx

    def traced():
        for grad in (False, True):
            x = torch.randn(3, 16, device=DEV, requires_grad=grad)
            for name, fn in operators(residual).items():
                with torch.set_grad_enabled(grad):
                    with pytest.raises(RuntimeError, match="cannot be traced"):
                        torch.jit.trace(fn, x, check_trace=False)
                    with pytest.raises(RuntimeError, match="cannot be traced"):
                        make_fx(fn)(x)
                    assert fn(x).shape == x.shape, name   # (and the next call is an ordinary one)
                if grad:
                    y = fn(x)
                    with pytest.raises(RuntimeError, match="cannot be traced"):
                        make_fx(lambda up: torch.autograd.grad(y, x, up))(torch.ones_like(y))
        state = residual.dropout_state(1, DEV)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda v: residual.take_dropout_state(state, 1), x.detach(), check_trace=False)
        none = torch.jit.trace(lambda v: residual.counter_dropout(v, 0.0, state), x.detach(), check_trace=False)
        assert torch.equal(none(2 * x.detach()), 2 * x)

    routes(traced)
