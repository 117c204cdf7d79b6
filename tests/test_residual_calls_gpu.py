"""The native host side of the residual-stream operators (host/residual_calls.cpp) against the Python route of residual.py."""
import gc
import random
import weakref

import pytest
import torch

import residual_oracle as ro
import test_residual_gpu as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def routes(monkeypatch):
    """Calls fn through the native host side and through the Python route."""
    from spiky_b200 import _native, residual

    native = _native.residual_calls()

    def both(fn):
        got = []
        for calls in (native, residual._PythonRoute):
            monkeypatch.setattr(residual, "_calls", calls)
            got.append(fn())
        return got

    return both


@pytest.mark.parametrize("seed", range(24))
def test_same_bits(routes, seed):
    rng = random.Random(seed)
    types = rng.choice(plain.TYPES)
    after, before = rng.choice([None, "rms", "layer"]), rng.choice([None, "rms", "layer"])
    alone = rng.random() < 0.2
    kw = dict(gate="none" if alone else rng.choice(["none", "one", "width", "sequence", "element"]), p=0.0 if alone else rng.choice([0.0, 0.2]),
              affine=rng.choice(["", "w", "wb"]), params=rng.choice([torch.float32, types[1]]), seed=seed, alone=alone, views=rng.random() < 0.3)
    lead, C = (rng.randrange(1, 6), rng.randrange(1, 40)), rng.choice([8, 61, 256, 1000])
    if alone:
        after, before = None, before or "rms"
    (out_a, grad_a), (out_b, grad_b) = routes(lambda: plain.run_join(*types, lead, C, after, before, **kw))
    for a, b in ((out_a, out_b), (grad_a, grad_b)):
        assert a.keys() == b.keys()
        for k in a:
            assert (a[k] is None and b[k] is None) or torch.equal(a[k], b[k]), k


def test_the_native_route_takes_ordinary_calls(monkeypatch):
    """Ordinary calls reach the native host side, forward and backward, and come back from it."""
    from spiky_b200 import _native, residual

    native, taken = _native.residual_calls(), []

    class Watch:
        pass

    for name in ("join", "dropout", "take"):
        def call(*args, _fn=getattr(native, name), _name=name):
            got = _fn(*args)
            taken.append((_name, got is not None))
            return got
        setattr(Watch, name, staticmethod(call))
    monkeypatch.setattr(residual, "_calls", Watch)
    state = residual.dropout_state(1, DEV)
    x, w = torch.randn(4, 3, 16, device=DEV, requires_grad=True), torch.nn.Parameter(torch.ones(16, device=DEV))
    used = residual.take_dropout_state(state, 1)
    h, y = residual.residual_join(x, x, branch_norm="layer", branch_weight=w, gate=w, dropout=0.5, state=used, next_norm="rms")
    z = residual.counter_dropout(residual.row_norm(y, w), 0.5, used)
    assert taken == [("take", True), ("join", True), ("join", True), ("dropout", True)]
    assert type(h.grad_fn).__name__ == "CppFunction" or "ResidualJoin" in h.grad_fn.name()
    (h.sum() + z.sum()).backward()
    assert x.grad is not None and w.grad is not None


def test_state_and_refusals(routes):
    routes(plain.test_state_moves_on_and_a_changed_state_is_refused)
    routes(plain.test_dropout_refusals)
    routes(plain.test_join_refusals)
    routes(plain.test_dropout_twice_differentiable)
    routes(lambda: [plain.test_no_rows(lead) for lead in ((0,), (3, 0), (0, 5))])
    routes(plain.test_dropout_edges)


def test_differentiable_once(routes):
    from spiky_b200 import residual

    def once():
        x = torch.randn(3, 16, device=DEV, requires_grad=True)
        y = residual.residual_join(x, x * 1, next_norm="rms")[1]
        g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            g.sum().backward()

    routes(once)


def test_inplace_change_is_seen(routes):
    from spiky_b200 import residual

    def changed():
        x = torch.randn(3, 16, device=DEV, requires_grad=True)
        f = torch.randn(3, 16, device=DEV)
        h = residual.residual_join(x, f, branch_norm="rms")
        f.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            h.sum().backward()

    routes(changed)


def test_contexts(routes):
    """no_grad, inference mode, a graph freed and used again, hooks on what is saved, functorch."""
    from spiky_b200 import residual

    def contexts():
        x, f = torch.randn(3, 16, device=DEV, requires_grad=True), torch.randn(3, 16, device=DEV)
        with torch.no_grad():
            assert residual.residual_join(x, f).grad_fn is None
        with torch.inference_mode():
            a = residual.residual_join(x, f, next_norm="rms")[1]
            assert a.is_inference()
        h = residual.residual_join(x, f, branch_norm="rms")
        h.sum().backward(retain_graph=True)
        h.sum().backward()
        with pytest.raises(RuntimeError, match="second time"):
            h.sum().backward()
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(1) or t.cpu(), lambda t: t.to(DEV)):
            h = residual.residual_join(x, f, branch_norm="rms")
        g, = torch.autograd.grad(h.sum(), x)
        assert packed and torch.equal(g, torch.ones_like(g))
        with pytest.raises(Exception):
            torch.func.vmap(lambda v: residual.row_norm(v))(torch.randn(2, 3, 16, device=DEV))
        return a.clone()

    a, b = routes(contexts)
    assert a.shape == b.shape


@pytest.mark.parametrize("kw,kept", [(dict(), 0), (dict(dropout=0.3), 0), (dict(gate="fixed"), 0), (dict(gate="learned"), 1), (dict(branch_norm="rms"), 1),
                                     (dict(next_norm="layer"), 2), (dict(branch_norm="rms", next_norm="rms", dropout=0.3, gate="learned"), 2)])
def test_what_is_kept_for_the_backward_pass(routes, kw, kept):
    """Tensors of the stream's size that a join keeps: none without norms and a learned gate; its gradients are right all the same."""
    from spiky_b200 import residual

    def run():
        for C in (64, 65, 16400):
            x, f = (torch.randn(4, 5, C, device=DEV, requires_grad=True) for _ in range(2))
            more = dict(kw)
            if "gate" in more:
                more["gate"] = torch.full((C,), 0.5, device=DEV, requires_grad=more["gate"] == "learned")
            if "dropout" in more:
                more["state"] = residual.dropout_state(2, DEV)
            seen = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.numel()) or t, lambda t: t):
                out = residual.residual_join(x, f, skip_scale=0.5, **more)
            assert seen.count(x.numel()) == kept
            if not kept:
                dh = torch.randn_like(x)
                dx, df = torch.autograd.grad(out, [x, f], dh)
                assert torch.equal(dx, 0.5 * dh)
                want = dh * 0.5 if "gate" in kw else dh
                if "dropout" in kw:
                    want = residual.counter_dropout(want, 0.3, more["state"])
                assert torch.equal(df, want)
            else:
                first = out if torch.is_tensor(out) else out[1]
                assert all(g.isfinite().all() for g in torch.autograd.grad(first.sum(), [x, f]))

    routes(run)


def test_what_hooks_hand_back_is_checked(routes):
    """A saved tensor that comes back on another device, of another type or size is an error, not an address for a kernel."""
    from spiky_b200 import residual

    def hooked():
        x, f = torch.randn(3, 16, device=DEV, requires_grad=True), torch.randn(3, 16, device=DEV)
        state = residual.dropout_state(1, DEV)
        for unpack in (lambda t: t, lambda t: t.to(DEV).double(), lambda t: t.to(DEV).reshape(-1)[:1]):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
                h = residual.residual_join(x, f, branch_norm="rms")
                y = residual.counter_dropout(x, 0.5, state)
            for out in (h, y):
                with pytest.raises(RuntimeError, match="forward pass"):
                    torch.autograd.grad(out.sum(), x)

    routes(hooked)


def test_lazily_negated_tensors(routes):
    from spiky_b200 import residual

    def negated():
        x = torch.randn(3, 16, device=DEV)
        n = torch._neg_view(x)
        state = residual.dropout_state(1, DEV)
        assert torch.equal(residual.residual_join(n, n), -2 * x)
        assert torch.equal(residual.counter_dropout(n, 0.5, state), -residual.counter_dropout(x, 0.5, state))
        w = torch.ones(16, device=DEV, requires_grad=True)
        y = residual.row_norm(n, w)
        g, = torch.autograd.grad(y, w, torch._neg_view(torch.ones_like(y)))
        ro.assert_near(g, residual.row_norm(x).sum(0).cpu().double(), torch.full((16,), 10.0, dtype=torch.float64), "dw")
        z = x.detach().requires_grad_()
        up = torch.randn_like(x)
        for out in (residual.residual_join(z, x, skip_scale=0.5), residual.counter_dropout(z, 0.5, state)):
            plain, = torch.autograd.grad(out, z, up, retain_graph=True)
            lazy, = torch.autograd.grad(out, z, torch._neg_view(up))
            assert torch.equal(lazy, -plain)

    routes(negated)


def test_graphs_are_freed(routes):
    from spiky_b200 import residual

    def freed():
        x = torch.randn(1024, 1024, device=DEV, requires_grad=True)
        gc.collect()   # (what other tests left)
        before = torch.cuda.memory_allocated()
        h, y = residual.residual_join(x, x * 1, branch_norm="rms", next_norm="rms")
        ref = weakref.ref(y)
        del h, y
        gc.collect()
        assert ref() is None and torch.cuda.memory_allocated() == before

    routes(freed)


def test_host_side_of_another_torch(monkeypatch):
    from spiky_b200 import _native, residual

    monkeypatch.setattr(residual, "_calls", None)
    monkeypatch.setattr(_native, "_residual_calls", None)
    monkeypatch.setattr(torch, "__version__", "1.2.3")
    x = torch.randn(3, 16, device=DEV)
    with pytest.warns(RuntimeWarning, match="Python route"):
        y = residual.row_norm(x)
    monkeypatch.undo()
    assert torch.equal(y, residual.row_norm(x))
