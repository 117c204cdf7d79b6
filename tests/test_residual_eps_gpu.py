"""Norms whose eps is not small beside the variance, and the first norm of a model: what a comparison at 1e-5 would not see."""
import pytest
import torch

import residual_oracle as ro
from test_residual_gpu import run_join
from test_transformer_joins_gpu import model, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("eps", [0.1, 3.0])
@pytest.mark.parametrize("C", [61, 256, 1000, 4096, 5003, 16384, 16400])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_eps_of_the_size_of_the_variance(eps, C, kind):
    """Every kernel's place for eps: beside the mean of squares, under the root, in both norms and in both directions."""
    run_join(F32, F32, (3, 5), C, None, kind, alone=True, eps=eps, seed=C)
    run_join(F32, F32, (3, 5), C, kind, kind, gate="width", p=0.2, eps=eps, seed=C)
    run_join(BF16, BF16, (3, 5), C, kind, None, eps=eps, seed=C)


def test_eps_of_the_modules():
    from spiky_b200 import residual

    x = torch.randn(4, 24, device=DEV)
    d = x.cpu().double()
    want = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 0.5)
    ro.assert_near(residual.RowNorm(24, eps=0.5, device=DEV)(x), want, 4 * want.abs() + 1, "RowNorm")
    h, y = residual.ResidualJoin(24, next_norm="rms", branch_scale=0.0, eps=0.5, device=DEV)(x, x)
    ro.assert_near(y, want, 4 * want.abs() + 1, "ResidualJoin")


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_first_norm_of_a_model(norm):
    """Its output and the gradients of its parameters, on the tensors that it met in the model."""
    m = model(norm=norm).train()
    with torch.no_grad():
        for p in m.first_norm.parameters():
            p.add_(0.1 * torch.randn(p.shape, generator=torch.Generator().manual_seed(4)).to(DEV))
    met = []

    def hook(module, args, out):
        out.retain_grad()
        met.append((args[0], out))

    m.first_norm.register_forward_hook(hook)
    logits = m(tokens())
    logits.backward(torch.randn(logits.shape, generator=torch.Generator().manual_seed(2)).to(DEV))
    (z, y), = met
    f = m.first_norm
    bias = None if f.bias is None else f.bias.detach().cpu().double()
    want = ro.join64(z.detach().cpu().double(), None, None, None, None, None, 1.0, 1.0, None, 1.0, norm, f.weight.detach().cpu().double(), bias, f.eps,
                     None, y.grad.cpu().double())
    ro.assert_near(y, *want["y"], "y")
    ro.assert_near(f.weight.grad, *want["dbw"], "weight")
    if f.bias is not None:
        ro.assert_near(f.bias.grad, *want["dbb"], "bias")


def test_transforms_raise():
    from spiky_b200 import residual

    x = torch.randn(2, 3, 16, device=DEV)
    state = residual.dropout_state(1, DEV)
    for fn in (lambda v: residual.row_norm(v), lambda v: residual.residual_join(v, v), lambda v: residual.counter_dropout(v, 0.5, state)):
        for call in (lambda: torch.func.vmap(fn)(x), lambda: torch.func.grad(lambda v: fn(v).sum())(x), lambda: torch.func.jvp(fn, (x,), (x,))):
            with pytest.raises(RuntimeError, match="functorch|data pointer|forward-mode"):
                call()
        assert fn(x).shape == x.shape
