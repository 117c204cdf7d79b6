"""Residual-stream operators under what torch does around a call - traces, recomputation, forward mode, second derivatives - on both routes."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_residual_calls_gpu import routes  # noqa: F401
from test_transformer_joins_gpu import model, tokens

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


# ------------------------------------------------------------------------------------------------ recomputation
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_dropout(routes, reentrant):  # noqa: F811
    """A state from outside gives both runs one mask; a state taken inside would be another one the second time, which is refused."""
    from spiky_b200 import residual
    from torch.utils.checkpoint import checkpoint

    def checkpointed():
        drop = residual.CounterDropout(0.5, seed=3, device=DEV)
        x = torch.randn(64, device=DEV, requires_grad=True)
        for part in (drop, lambda v: residual.counter_dropout(v, 0.5, residual.take_dropout_state(drop.state, 1))):
            y = checkpoint(part, x, use_reentrant=reentrant)
            with pytest.raises(RuntimeError, match="outside the part that is run again"):
                y.sum().backward()
        drop.load_state_dict({"state": residual.dropout_state(3, "cpu")})
        want = drop(x)
        dwant, = torch.autograd.grad((want * want).sum(), x)
        drop.load_state_dict({"state": residual.dropout_state(3, "cpu")})
        x.grad = None
        y = checkpoint(lambda v, s: drop(v, s) ** 2, x, drop.take_state(), use_reentrant=reentrant)
        y.sum().backward()
        assert torch.equal(y, want * want) and torch.equal(x.grad, dwant)
        assert drop.state.tolist() == [3, 1]
        assert torch.equal(drop.eval()(x, drop.take_state()), x)

    routes(checkpointed)


@pytest.mark.parametrize("opts", [dict(), dict(use_batch_norm=True), dict(norm="rms", gated=True)])
def test_checkpointed_model(opts):
    """A whole model run again in the backward pass (table gradients are summed by atomics)."""
    from torch.utils.checkpoint import checkpoint

    start = model(dropout=0.4, counter_dropout=True, **opts).state_dict()   # (a seed is that of anchors and embeddings, not of the tables)

    def gradients(call):
        m = model(dropout=0.4, counter_dropout=True, **opts).train()
        m.load_state_dict(start)
        params = [p for p in m.parameters() if p.requires_grad]
        out = call(m)
        dl = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(DEV)
        out.backward(dl)
        assert m.dropout_state.tolist() == [7, m._n_dropouts]
        return out, [p.grad for p in params]

    want, dwant = gradients(lambda m: m(tokens()))
    got, dgot = gradients(lambda m: checkpoint(m, tokens(), m.take_dropout_state(), use_reentrant=False))
    assert torch.equal(got, want)
    for a, b in zip(dgot, dwant):
        assert (a - b).abs().max() <= 1e-5 * b.abs().max() + 1e-12
    m = model(dropout=0.4, counter_dropout=True, **opts).train()
    out = checkpoint(m, tokens(), use_reentrant=False)
    with pytest.raises(RuntimeError, match="outside the part that is run again"):
        out.sum().backward()
    m.eval()
    state = m.train().take_dropout_state()
    assert m.eval().take_dropout_state() is None and torch.equal(m(tokens(), state), m(tokens()))
    with pytest.raises(ValueError, match="counter_dropout"):
        model(dropout=0.4)(tokens(), state)


# ------------------------------------------------------------------------------------------------ forward mode
def test_forward_mode_is_refused(routes):  # noqa: F811
    """A tangent is not dropped in silence: dual inputs that want no gradient, dual parameters, dual gradients."""
    from spiky_b200 import residual

    def dual_calls():
        x, w = torch.randn(3, 16, device=DEV), torch.ones(16, device=DEV)
        with forward_ad.dual_level():
            d, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
            calls = [lambda fn=fn: fn(d) for fn in operators(residual).values()]
            calls += [lambda: residual.row_norm(x, dw), lambda: residual.row_norm(x, w, dw), lambda: residual.residual_join(x, d),
                      lambda: residual.residual_join(x, x, gate=dw), lambda: residual.residual_join(x, x, gate=dw[:1]), lambda: residual.row_norm(d[:0]),
                      lambda: residual.residual_join(x, x, branch_norm="rms", branch_weight=dw)]
            for call in calls:
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
            assert torch.equal(forward_ad.unpack_dual(residual.counter_dropout(d, 0.0, None)).tangent, torch.ones_like(x))
            assert residual.row_norm(x, w).shape == x.shape   # (a level without tangents is an ordinary one)
            for fn in operators(residual).values():
                z = x.clone().requires_grad_()
                y = fn(z)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch.autograd.grad(y, z, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))

    routes(dual_calls)


# ------------------------------------------------------------------------------------------------ second derivatives
def test_second_derivatives_are_not_left_out(routes):  # noqa: F811
    """A penalty on a gradient raises, whether the incoming gradient wants one (y * y) or is a constant (a plain sum), whichever way it is asked."""
    from spiky_b200 import residual
    from torch.utils.checkpoint import checkpoint

    def penalties():
        def leaf(*shape):
            return torch.randn(*shape, device=DEV, requires_grad=True)

        def raises(loss, of):
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(loss, of, retain_graph=True)
            with pytest.raises(RuntimeError, match="differentiable once"):
                loss.backward()

        x, f, gate, w, b = leaf(3, 16), leaf(3, 16), leaf(16), leaf(16), leaf(16)
        for fn in (lambda: residual.row_norm(x, w, b), lambda: residual.residual_join(x, f, gate=gate, next_norm="layer", next_weight=w, next_bias=b)[1]):
            for loss in (lambda y: y.sum(), lambda y: (y * y).sum()):
                g, = torch.autograd.grad(loss(fn()), x, create_graph=True)
                raises(x.sum() + (g * g).sum(), x)
                g, = torch.autograd.grad(loss(fn()), w, create_graph=True)
                raises(w.sum() + g.sum(), [w, x])
        # a join without the next norm: what does not depend on an input stays an ordinary constant
        h = residual.residual_join(x, f, branch_norm="rms", branch_weight=w, branch_bias=b, gate=gate, skip_scale=0.5)
        for name, t, of in (("branch", f, f), ("branch by weight", f, w), ("branch by gate", f, gate), ("gate", gate, b), ("weight", w, gate), ("bias", b, gate)):
            g, = torch.autograd.grad(h.sum(), t, create_graph=True)
            raises(of.sum() + g.sum(), of)
        g, = torch.autograd.grad(h.sum(), x, create_graph=True)
        assert not g.requires_grad and torch.equal(g, torch.full_like(g, 0.5))
        y = residual.row_norm(x, w, b)
        g, = torch.autograd.grad(y.sum(), b, create_graph=True)
        assert not g.requires_grad and torch.equal(g, torch.full_like(g, 3.0))
        # the gradients themselves are those without a graph, and so is a sum of ordinary terms
        up = torch.randn(3, 16, device=DEV)
        plain = torch.autograd.grad(h, [x, f, gate, w, b], up, retain_graph=True)
        graphed = torch.autograd.grad(h, [x, f, gate, w, b], up, create_graph=True)
        assert all(torch.equal(p, g) for p, g in zip(plain, graphed))
        x.grad = None
        (x.sum() + residual.row_norm(x).sum()).backward(create_graph=True)
        assert x.grad.requires_grad
        x.grad = None
        # a join that is run again, with a graph of its gradient
        fn = lambda v: residual.residual_join(v, v * 2, branch_norm="rms", gate=gate[:1], next_norm="layer")[1]  # noqa: E731
        g, = torch.autograd.grad(checkpoint(fn, x, use_reentrant=False), x, up, create_graph=True)
        want, = torch.autograd.grad(fn(x), x, up)
        assert torch.equal(g, want)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum(), x)

    routes(penalties)


# ------------------------------------------------------------------------------------------------ compiled functions
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_calls_in_compiled_functions(routes, backend):  # noqa: F811
    """torch.compile runs the calls between its graphs, on either route, on the stream that is current when they run."""
    from spiky_b200 import residual

    def compiled():
        gate, state = torch.full((1,), 0.5, device=DEV), residual.dropout_state(1, DEV)
        calls = [lambda v: residual.residual_join(v, v * 2, gate=gate) * 2, lambda v: residual.residual_join(v, v, next_norm="rms")[1] + v,
                 lambda v: residual.counter_dropout(v, 0.5, state) + v, lambda v: residual.row_norm(v) * v]
        for fn in calls:
            torch._dynamo.reset()
            x = torch.randn(5, 16, device=DEV)
            quick = torch.compile(fn, backend=backend)
            assert torch.equal(quick(x), fn(x))
            z = x.clone().requires_grad_()
            got, want = (torch.autograd.grad(f(z).sum(), z)[0] for f in (quick, fn))
            assert torch.equal(got, want)
            graph = torch.cuda.CUDAGraph()
            with torch.no_grad(), torch.cuda.graph(graph):
                out = quick(x)
            x.normal_()
            graph.replay()
            assert torch.equal(out, fn(x))

    routes(compiled)
    torch._dynamo.reset()
