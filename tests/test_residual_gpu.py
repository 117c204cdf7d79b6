"""Dropout without a stored mask, row norms and residual joins on the GPU against their 64-bit statements (residual_oracle)."""
import random

import pytest
import torch

import residual_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.bfloat16),
         (torch.float32, torch.float16)]
IDS = ["f32", "bf16", "f16", "f32-bf16", "f32-f16"]


def lib():
    from spiky_b200 import residual
    return residual


def normal(gen, shape, scale=1.0, mean=0.0):
    return mean + scale * torch.randn(shape, generator=gen)


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 31, 256, 4099, 100003])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout(dtype, n, p):
    gen = torch.Generator().manual_seed(n)
    seed, offset, site = 0x123456789ABCDEF0 - n, 2 ** 32 - 2, 5   # (the offset carries into its upper half)
    state = lib().dropout_state(seed, DEV, offset)
    x = normal(gen, (n,)).to(dtype).to(DEV).requires_grad_()
    dy = normal(gen, (n,)).to(dtype).to(DEV)
    y = lib().counter_dropout(x, p, state, site)
    kept = ro.keeps(p, seed, offset + site, n)
    dx, = torch.autograd.grad(y, x, dy)
    for got, of in ((y, x), (dx, dy)):
        want = torch.where(kept, of.detach().cpu().double() * ro.drop_scale(p), 0.0)
        assert got.dtype == dtype
        ro.assert_near(got, want, want.abs(), "dropout")
        assert torch.equal(got.detach().cpu() == 0, ~kept | (of.detach().cpu() == 0))
    assert torch.equal(y, lib().counter_dropout(x.detach(), p, state, site))


def test_dropout_ties_take_the_second_digit():
    """Thresholds chosen at the numbers of drawn elements: an element whose number is the threshold stays, one below goes."""
    seed, offset, n = 99, 3, 4096
    u = ro.numbers(seed, offset, 0, n)
    state = lib().dropout_state(seed, DEV, offset)
    x = torch.ones(n, device=DEV)
    for i in (0, 1, 6, 7, 100, 4095):
        for t in (int(u[i]), int(u[i]) + 1, int(u[i]) & ~0xFFFF, (int(u[i]) | 0xFFFF) + 1):
            p = t / 2.0 ** 32
            assert ro.threshold(p) == t
            y = lib().counter_dropout(x, p, state)
            assert torch.equal(y.cpu() != 0, torch.from_numpy(u >= t) & (t < 2 ** 32)), (i, t)


def test_dropout_edges():
    state = lib().dropout_state(1, DEV)
    x = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0] * 500, device=DEV)
    y = lib().counter_dropout(x, 0.5, state)
    kept = ro.keeps(0.5, 1, 0, 2000).to(DEV)
    assert torch.all(y[~kept] == 0) and torch.equal(y[kept].isnan(), x[kept].isnan()) and torch.equal(y[kept].isinf(), x[kept].isinf())
    assert torch.all(lib().counter_dropout(x, 1.0, state) == 0)
    same = lib().counter_dropout(x, 0.0, None)
    assert torch.equal(same.nan_to_num(), x.nan_to_num()) and same.data_ptr() != x.data_ptr()
    one = x[3:4].expand(100)
    assert torch.equal(lib().counter_dropout(one, 1e-12, state), one)   # (below half a step of the threshold)
    assert lib().counter_dropout(x[:0], 0.5, state).shape == (0,)
    # views: misaligned, strided, transposed; numbered by their own elements
    base = torch.randn(70, 33, device=DEV).bfloat16()
    for v in (base.reshape(-1)[1:], base[:, 1:], base.t(), base[::2, ::3]):
        flat = lib().counter_dropout(v.contiguous().clone(), 0.3, state)
        assert torch.equal(lib().counter_dropout(v, 0.3, state), flat)


def test_dropout_beyond_32_bits():
    n, tail = 2 ** 32 + 12345, 5000
    state = lib().dropout_state(7, DEV, 11)
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    y = lib().counter_dropout(x, 0.5, state)
    for first in (0, 2 ** 31 - 100, 2 ** 32 - 100, n - tail):
        assert torch.equal(y[first:first + tail].cpu() != 0, ro.keeps(0.5, 7, 11, tail, first)), first


def test_dropout_refusals():
    r = lib()
    x, state = torch.zeros(4, 8, device=DEV), r.dropout_state(1, DEV)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            r.counter_dropout(x, p, state)
    with pytest.raises(ValueError):
        r.counter_dropout(x, 0.5, state, site=-1)
    for bad in (None, torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), state.cpu()):
        with pytest.raises(RuntimeError):
            r.counter_dropout(x, 0.5, bad)
    for bad in (x.double(), x.long(), x.cpu(), x.to_sparse()):
        with pytest.raises(RuntimeError):
            r.counter_dropout(bad, 0.5, state)


def test_state_moves_on_and_a_changed_state_is_refused():
    r = lib()
    state = r.dropout_state(5, DEV, -1)
    first, second = r.take_dropout_state(state, 3), r.take_dropout_state(state, 4)
    assert first.tolist() == [5, -1] and second.tolist() == [5, 2] and state.tolist() == [5, 6]
    x = torch.randn(64, device=DEV, requires_grad=True)
    y = r.counter_dropout(x, 0.5, state)
    r.take_dropout_state(state, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_twice_differentiable():
    r = lib()
    state = r.dropout_state(5, DEV)
    x = torch.randn(640, device=DEV, requires_grad=True)
    y = r.counter_dropout(x, 0.5, state)
    dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    ddx, = torch.autograd.grad(dx.sum(), x)
    kept = ro.keeps(0.5, 5, 0, 640).to(DEV)
    assert torch.equal(ddx, torch.where(kept, 8.0, 0.0))


# ------------------------------------------------------------------------------------------------ joins and norms
def run_join(stream, branch, lead, C, after, before, gate="none", p=0.0, affine="wb", params=None, skip=0.75, scale=0.5, eps=1e-5, seed=0,
             ups="hy", alone=False, mean=0.3, views=False):
    """One join (or, alone, a norm) forward and backward against join64."""
    r, gen = lib(), torch.Generator().manual_seed(1000 + seed)
    shape = tuple(lead) + (C,)
    params = params or torch.float32

    def leaf(shape, dtype, s=1.0, m=0.0, view=False):
        t = normal(gen, shape, s, m).to(dtype).to(DEV)
        if view:   # the same values behind other strides and an odd start
            wide = torch.empty(tuple(t.shape[:-1]) + (t.shape[-1] + 3,), dtype=dtype, device=DEV)
            wide[..., 1:-2] = t
            t = wide[..., 1:-2]
        return t.detach().requires_grad_()

    v = dict(x=leaf(shape, stream, 1.0, mean, views))
    if not alone:
        v["f"] = leaf(shape, branch, 0.7, 0.1, views)
    if gate != "none":
        v["gate"] = leaf({"one": (1,), "width": (C,), "sequence": (lead[0],) + (1,) * (len(lead) - 1) + (C,), "element": shape}[gate],
                         branch if gate == "element" else params, 0.3, 0.8)
    for name, kind in (("a", after), ("b", before)):
        if kind:
            if "w" in affine:
                v[name + "w"] = leaf((C,), params, 0.2, 1.0)
            if "b" in affine:
                v[name + "b"] = leaf((C,), params, 0.3)
    up = {}
    if not alone and "h" in ups:
        up["h"] = normal(gen, shape).to(stream).to(DEV)
    if before and "y" in ups:
        up["y"] = normal(gen, shape).to(branch).to(DEV)
    rseed, offset, site = 77 + seed, 2 ** 40 + seed, seed % 3
    state = r.dropout_state(rseed, DEV, offset) if p else None

    def call(v):
        if alone:
            return dict(y=r.row_norm(v["x"], v.get("bw"), v.get("bb"), kind=before, eps=eps, dtype=branch))
        got = r.residual_join(v["x"], v["f"], branch_norm=after, branch_weight=v.get("aw"), branch_bias=v.get("ab"), gate=v.get("gate"),
                              skip_scale=skip, branch_scale=scale, dropout=p, state=state, site=site, next_norm=before,
                              next_weight=v.get("bw"), next_bias=v.get("bb"), eps=eps)
        return dict(h=got) if before is None else dict(h=got[0], y=got[1])

    out = call(v)
    names = list(v)
    grads = torch.autograd.grad([out[k] for k in up], [v[k] for k in names], [up[k] for k in up], allow_unused=True)
    d = {k: t.detach().cpu().double() for k, t in v.items()}
    n = v["x"].numel()
    kept = ro.keeps(p, rseed, offset + site, n).view(shape) if p else None
    want = ro.join64(d["x"], d.get("f"), after, d.get("aw"), d.get("ab"), d.get("gate"), skip, scale, kept, ro.drop_scale(p), before, d.get("bw"),
                     d.get("bb"), eps, *(up[k].cpu().double() if k in up else None for k in "hy"))
    types = dict(h=stream, y=branch)
    for k, t in out.items():
        assert t.dtype == types[k]
        ro.assert_near(t, *want[k], k)
    for k, g in zip(names, grads):
        if g is None:
            assert k in ("bw", "bb") and "y" not in up, k
            continue
        assert g.dtype == v[k].dtype, k
        ro.assert_near(g, *want["d" + k], "d" + k)
    again = call({k: t.detach() for k, t in v.items()})   # without a graph: the same values
    for k in out:
        assert torch.equal(out[k], again[k])
    more = torch.autograd.grad(list(call(v).values())[0].float().sum(), [v["x"]])   # (and a second backward pass of a new graph runs)
    assert more[0].shape == shape
    return out, dict(zip(names, grads))


WIDTHS = [1, 2, 7, 8, 24, 64, 65, 250, 256, 257, 1000, 1024, 1031, 2048, 2056, 4096, 4100, 8192]


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("C", WIDTHS)
def test_join_widths(types, C):
    rng = random.Random(C)
    run_join(*types, (3, 5), C, rng.choice(["rms", "layer"]), rng.choice(["rms", "layer"]), gate=rng.choice(["none", "width", "sequence", "element"]),
             p=0.2, params=rng.choice([torch.float32, types[1]]), seed=C)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]], ids=["f32", "f32-bf16"])
@pytest.mark.parametrize("C", [2049, 2600, 3001, 4104, 8184, 8193, 12000, 12001, 16383, 16384])
def test_join_wide_rows(types, C):
    """Blocks of 512 threads and clusters, of whole groups and of odd rows; each sum, and more rows than are taken at once."""
    run_join(*types, (2, 3), C, "layer", "layer", gate="sequence", p=0.1, seed=C)
    run_join(*types, (170, 1), C, "rms", "rms", gate="width", p=0.3, seed=C + 1, params=types[1])
    run_join(*types, (2, 2), C, None, "layer", alone=True, seed=C)


@pytest.mark.parametrize("after", [None, "rms", "layer"])
@pytest.mark.parametrize("before", [None, "rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "one", "width", "sequence", "element"])
@pytest.mark.parametrize("C", [48, 52])
def test_join_forms(after, before, gate, C):
    rng = random.Random(str((after, before, gate, C)))
    run_join(*rng.choice(TYPES), (4, 9), C, after, before, gate=gate, p=rng.choice([0.0, 0.3]), affine=rng.choice(["", "w", "b", "wb"]), seed=C)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("C", [1, 16, 100, 256, 1024, 1027, 4096])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norms(types, C, kind):
    run_join(*types, (2, 33), C, None, kind, alone=True, seed=C, mean=0.5)


@pytest.mark.parametrize("lead,gate", [((1,), "width"), ((2, 700), "sequence"), ((700, 2), "sequence"), ((3, 1, 411), "sequence"), ((5000,), "width"),
                                       ((61, 67), "none"), ((1, 1), "element"), ((30000,), "none")])
@pytest.mark.parametrize("C", [32, 33])
def test_join_rows(lead, gate, C):
    """Row counts from one to more than the blocks take at once; groups of rows with a gate row of their own, few and many."""
    run_join(torch.float32, torch.float32, lead, C, "layer", "rms", gate=gate, p=0.1, seed=len(lead))
    run_join(torch.float32, torch.bfloat16, lead, C, None, "layer", gate=gate, seed=len(lead))


@pytest.mark.parametrize("C,lead", [(1024, (2600,)), (256, (64, 128)), (4096, (700,)), (1000, (2100,))])
def test_join_many_rows(C, lead):
    run_join(torch.bfloat16, torch.bfloat16, lead, C, "rms", "layer", gate="width", p=0.1, seed=C)


@pytest.mark.parametrize("C", [8200, 10001, 20000])
def test_join_very_wide(C):
    run_join(torch.float32, torch.bfloat16, (3,), C, "layer", "rms", gate="width", p=0.1, seed=C)
    run_join(torch.float32, torch.float32, (5,), C, None, "layer", alone=True, seed=C)
    if C == 20000:   # more gate rows than blocks, fewer, and one in pieces
        run_join(torch.float32, torch.float32, (700, 2), C, "rms", None, gate="sequence", seed=1)
        run_join(torch.bfloat16, torch.bfloat16, (3, 40), C, None, "rms", gate="sequence", params=torch.bfloat16, seed=2)
        run_join(torch.float32, torch.float32, (900,), C, None, None, gate="width", seed=3)


@pytest.mark.parametrize("ups", ["h", "y", "hy"])
@pytest.mark.parametrize("C", [64, 67])
def test_join_one_gradient(ups, C):
    run_join(torch.float32, torch.float32, (3, 4), C, "layer", "layer", gate="width", p=0.2, ups=ups, seed=3)
    run_join(torch.bfloat16, torch.bfloat16, (3, 4), C, None, "rms", ups=ups, seed=4)


@pytest.mark.parametrize("C", [64, 1024, 67])
def test_join_of_views(C):
    run_join(torch.bfloat16, torch.bfloat16, (6, 4), C, "rms", "rms", gate="element", p=0.2, views=True, seed=5)
    run_join(torch.float32, torch.float32, (6, 4), C, None, "layer", gate="sequence", views=True, seed=6)
    # contiguous, but not on a 16-byte boundary
    r, gen = lib(), torch.Generator().manual_seed(9)
    flat = normal(gen, (2, 5 * C + 1)).bfloat16().to(DEV)
    x, f = flat[0, 1:].view(5, C), flat[1, 1:].view(5, C)
    for got, want in zip(r.residual_join(x, f, next_norm="rms"), r.residual_join(x.clone(), f.clone(), next_norm="rms")):
        ro.assert_near(got, want.cpu().double(), want.cpu().double().abs() + 1, "misaligned")


@pytest.mark.parametrize("C", [64, 67])
def test_rows_that_are_dropped_whole(C):
    """With p = 1 the branch is zeros: its norm is of a row of zeros, the result its bias, the gradient zero."""
    r = lib()
    state = r.dropout_state(1, DEV)
    x = torch.randn(4, C, device=DEV)
    f = torch.full((4, C), float("nan"), device=DEV, requires_grad=True)
    bias = torch.randn(C, device=DEV)
    for kind in ("rms", "layer"):
        h = r.residual_join(x, f, branch_norm=kind, branch_bias=bias, dropout=1.0, state=state)
        assert torch.equal(h, x + bias)
        df, = torch.autograd.grad(h.sum(), f)
        assert torch.all(df == 0)
    h = r.residual_join(x, f, dropout=1.0, state=state)
    assert torch.equal(h, x)


def test_rows_of_one_value():
    """A constant row has no deviation: its layer norm is the bias, and finite gradients."""
    r = lib()
    x = torch.full((3, 40), 2.5, device=DEV, requires_grad=True)
    bias = torch.randn(40, device=DEV)
    y = r.row_norm(x, None, bias, kind="layer")
    assert torch.equal(y, bias.expand(3, 40))
    dx, = torch.autograd.grad(y, x, torch.randn(3, 40, device=DEV))
    assert dx.isfinite().all()


def test_bad_values_stay_in_their_row():
    r = lib()
    for C in (256, 100):
        x, f = torch.randn(6, C, device=DEV), torch.randn(6, C, device=DEV)
        f[2, 5], x[4, 7] = float("nan"), float("inf")
        h, y = r.residual_join(x, f, branch_norm="layer", next_norm="rms")
        good = torch.tensor([0, 1, 3, 5], device=DEV)
        h2, y2 = r.residual_join(x[good], f[good], branch_norm="layer", next_norm="rms")
        assert torch.equal(h[good], h2) and torch.equal(y[good], y2)
        assert h[2].isnan().all() and y[2].isnan().all() and h[4, 7].isinf()


@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 5)])
def test_no_rows(lead):
    r = lib()
    x = torch.zeros(*lead, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    gates = [None, torch.ones(16, device=DEV, requires_grad=True)]
    if len(lead) == 2:
        gates.append(torch.ones(lead[0], 1, 16, device=DEV, requires_grad=True))
    for gate in gates:
        h, y = r.residual_join(x, x * 1, branch_norm="rms", branch_weight=w, gate=gate, next_norm="layer", next_weight=w, dropout=0.5,
                               state=r.dropout_state(1, DEV))
        assert h.shape == x.shape and y.shape == x.shape
        (h.sum() + y.sum()).backward()
        assert torch.all(w.grad == 0) and x.grad.shape == x.shape
        assert gate is None or torch.all(gate.grad == 0)
    assert r.row_norm(x).shape == x.shape


def test_the_join_is_its_parts():
    """Dropout inside a join is counter_dropout of the branch; the next norm is that of the sum."""
    r = lib()
    for C in (96, 101):
        x, f, w = torch.randn(7, 9, C, device=DEV), torch.randn(7, 9, C, device=DEV), torch.rand(C, device=DEV)
        state = r.dropout_state(3, DEV, 10)
        h, y = r.residual_join(x, f, dropout=0.4, state=state, site=2, next_norm="rms", next_weight=w)
        assert torch.equal(h, x + r.counter_dropout(f, 0.4, state, 2))
        ro.assert_near(y, r.row_norm(h, w).cpu().double(), y.cpu().double().abs() + 1e-3, "y")


def test_two_calls_the_same_bits():
    for C in (256, 250):
        one = run_join(torch.float32, torch.float32, (40, 33), C, "layer", "rms", gate="sequence", p=0.1, seed=8)
        two = run_join(torch.float32, torch.float32, (40, 33), C, "layer", "rms", gate="sequence", p=0.1, seed=8)
        for a, b in zip(one, two):
            for k in a:
                assert torch.equal(a[k], b[k]), k


def test_join_refusals():
    r = lib()
    x, w = torch.zeros(2, 3, 8, device=DEV), torch.ones(8, device=DEV)
    for kw in (dict(branch_norm="batch"), dict(next_norm="l2"), dict(branch_weight=w), dict(next_bias=w), dict(next_norm="rms", next_weight=w[:4]),
               dict(gate=torch.ones(4, device=DEV)), dict(gate=torch.ones(3, 8, device=DEV)), dict(gate=torch.ones(1, 3, 1, device=DEV)), dict(eps=0.0),
               dict(eps=1e-60), dict(eps=float("nan")), dict(skip_scale=float("nan")), dict(branch_scale=float("inf")), dict(dropout=1.5), dict(site=-1)):
        with pytest.raises(ValueError):
            r.residual_join(x, x, **kw)
    for kw in (dict(next_norm="rms", next_weight=w.bfloat16()), dict(next_norm="rms", next_weight=w.cpu()), dict(gate=w.half()), dict(dropout=0.5),
               dict(next_norm="rms", branch_norm="rms", next_weight=w, branch_weight=w.double())):
        with pytest.raises(RuntimeError):
            r.residual_join(x, x, **kw)
    xb = x.bfloat16()
    with pytest.raises(RuntimeError, match="one type"):
        r.residual_join(xb, xb, branch_norm="rms", next_norm="rms", branch_weight=w, next_weight=w.bfloat16())
    for a, b in ((xb, x), (xb, x.half()), (x, x.double()), (x.cpu(), x), (x, x.cpu())):
        with pytest.raises(RuntimeError):
            r.residual_join(a, b)
    with pytest.raises(ValueError):
        r.residual_join(x, x[:1])
    with pytest.raises(ValueError):
        r.row_norm(torch.zeros((), device=DEV))
    with pytest.raises(ValueError):
        r.row_norm(torch.zeros(3, 0, device=DEV))
    with pytest.raises(ValueError):
        r.row_norm(x, kind=None)
    with pytest.raises(RuntimeError):
        r.row_norm(xb, dtype=torch.float32)
    y = r.row_norm(x.requires_grad_())
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_join_beyond_32_bits():
    """More than 2^31 elements: the last rows are what they are alone."""
    r, C = lib(), 2048
    rows = 2 ** 31 // C + 37
    x = torch.empty(rows, C, dtype=torch.bfloat16, device=DEV)
    f = torch.empty(rows, C, dtype=torch.bfloat16, device=DEV)
    x.normal_()
    f.normal_()
    h, y = r.residual_join(x, f, branch_norm="rms", next_norm="layer")
    some = torch.tensor([0, rows // 2, rows - 2, rows - 1], device=DEV)
    h2, y2 = r.residual_join(x[some], f[some], branch_norm="rms", next_norm="layer")
    assert torch.equal(h[some], h2) and torch.equal(y[some], y2)
    del h, y
    x.requires_grad_()
    y = r.row_norm(x)
    dx, = torch.autograd.grad(y, x, f)
    x2 = x.detach()[some].requires_grad_()
    dx2, = torch.autograd.grad(r.row_norm(x2), x2, f[some])
    assert torch.equal(dx[some], dx2)


def test_more_rows_than_32_bit_numbers_of_the_row_kernels():
    r, rows = lib(), 2 ** 30 + 3
    x = torch.empty(rows, 1, dtype=torch.float16, device=DEV).normal_()
    h = r.residual_join(x, x, branch_scale=0.5)
    for part in (slice(0, 1000), slice(rows - 1000, rows)):
        ro.assert_near(h[part], 1.5 * x[part].cpu().double(), 1.5 * x[part].cpu().double().abs(), "h")


def test_no_wait_of_a_cluster_ran_out():
    from spiky_b200 import _native

    run_join(torch.float32, torch.float32, (300,), 16384, "layer", "layer", gate="width", p=0.1, seed=1)
    assert _native.device_wait_errors() == 0


def test_side_stream_and_graph():
    """A training pass on a stream of its own, captured and replayed: each replay moves the dropout on and uses new inputs."""
    r = lib()
    x, f, w = torch.randn(50, 64, device=DEV), torch.randn(50, 64, device=DEV), torch.rand(64, device=DEV)
    g = torch.randn(50, 64, device=DEV)
    state = r.dropout_state(21, DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, f, w)]
        used = r.take_dropout_state(state, 2)
        h, y = r.residual_join(leaves[0], leaves[1], dropout=0.3, state=used, site=1, next_norm="rms", next_weight=leaves[2])
        z = r.counter_dropout(y, 0.5, used, site=0)
        return [h, y, z] + list(torch.autograd.grad([h, z], leaves, [g, g]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [[t.detach().clone() for t in step()] for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    state.copy_(r.dropout_state(21, DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    state.copy_(r.dropout_state(21, DEV))
    for want in eager:
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    assert state.tolist() == [21, 6]
    x.mul_(2.0)
    graph.replay()
    changed = [t.detach().clone() for t in out]
    state.copy_(r.dropout_state(21, DEV, 6))
    for a, b in zip(changed, step()):
        assert torch.equal(a, b)


def test_modules():
    r = lib()
    drop = r.CounterDropout(0.25, seed=4, device=DEV)
    x = torch.randn(5, 24, device=DEV)
    one, two = drop(x), drop(x)
    assert not torch.equal(one, two) and drop.state.tolist() == [4, 2]
    drop.load_state_dict({"state": r.dropout_state(4, "cpu")})
    assert torch.equal(drop(x), one)
    assert drop.eval()(x) is x
    norm = r.RowNorm(24, "layer", device=DEV)
    ro.assert_near(norm(x), torch.nn.functional.layer_norm(x.cpu().double(), (24,), eps=1e-6), x.cpu().double().abs() + 1, "norm")
    join = r.ResidualJoin(24, "rms", "layer", gated=True, gate_init=0.5, dropout=0.5, device=DEV)
    state = r.dropout_state(1, DEV)
    h, y = join(x, x, state, 3)
    (h.sum() + (y * y).sum()).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in join.parameters())
    h, y = join.eval()(x, x)
    assert torch.equal(h, r.residual_join(x, x, branch_norm="rms", gate=join.gate, next_norm=None))
    plain = r.ResidualJoin(24, device=DEV)
    h, y = plain(x, x)
    assert h is y and torch.equal(h, x + x)


@pytest.mark.parametrize("C,shift", [(64, 0), (64, 1), (67, 0), (67, 3), (1024, 2), (1031, 0), (5000, 0), (5001, 1), (16400, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_nothing_beside_the_outputs_is_written(C, shift, dtype):
    """The C entry points on arrays that begin anywhere, each between guards: the results are those of aligned arrays, the guards stay."""
    import ctypes

    from spiky_b200 import _native as nat

    L, gen, rows, GUARD = nat.lib(), torch.Generator().manual_seed(C), 7, 64
    code = nat.F32 if dtype == torch.float32 else nat.BF16
    values = {k: normal(gen, s).to(dtype).to(DEV) for k, s in dict(x=(rows, C), f=(rows, C), gate=(rows, C), aw=(C,), ab=(C,), bw=(C,), bb=(C,),
                                                                   dh=(rows, C), dy=(rows, C)).items()}
    state = lib().dropout_state(3, DEV)
    cfg = nat.JoinCfg(rows=rows, width=C, gate_rows=1, site=1, dropout=0.25, stream_type=code, branch_type=code, param_type=code, gate_type=code,
                      after=nat.NORM_LAYER, before=nat.NORM_RMS, eps=1e-5, skip_scale=0.5, branch_scale=2.0)
    stream = torch.cuda.current_stream().cuda_stream

    def run(shift):
        held, outs = [], {}

        def placed(t, guard):
            flat = torch.full((t.numel() + shift + GUARD,), guard, dtype=t.dtype, device=DEV)
            flat[shift:shift + t.numel()] = t.reshape(-1)
            held.append(flat)
            return flat[shift:shift + t.numel()]

        v = {k: placed(t, float("nan")) for k, t in values.items()}   # (what is beside an input may be read, never used)

        def out(name, *shape):
            flat = torch.full((torch.Size(shape).numel() + 2 * GUARD + shift,), 7.0, dtype=dtype, device=DEV)
            outs[name] = flat
            return flat.data_ptr() + (GUARD + shift) * flat.element_size()

        stats = torch.zeros(rows, 4, device=DEV)
        p = {k: t.data_ptr() for k, t in v.items()}
        nat.check(L.lutb_join_forward(ctypes.byref(cfg), p["x"], p["f"], p["gate"], p["aw"], p["ab"], p["bw"], p["bb"], state.data_ptr(),
                                      out("h", rows, C), out("y", rows, C), stats.data_ptr(), stream))
        need = L.lutb_join_backward_workspace(ctypes.byref(cfg))
        ws = torch.full((need + 64,), 9, dtype=torch.uint8, device=DEV)
        nat.check(L.lutb_join_backward(ctypes.byref(cfg), p["x"], p["f"], p["gate"], p["aw"], p["ab"], p["bw"], state.data_ptr(), stats.data_ptr(), p["dh"],
                                       p["dy"], out("dx", rows, C), out("df", rows, C), out("dgate", rows, C), out("daw", C), out("dab", C),
                                       out("dbw", C), out("dbb", C), ws.data_ptr(), need, stream))
        nat.check(L.lutb_dropout(code, rows * C, 0.25, state.data_ptr(), 0, p["x"], out("z", rows, C), stream))
        torch.cuda.synchronize()
        assert torch.all(ws[need:] == 9)
        got = {}
        for name, flat in outs.items():
            inner = flat[GUARD + shift:-GUARD]
            assert torch.all(flat[:GUARD + shift] == 7) and torch.all(flat[-GUARD:] == 7), name
            got[name] = inner.clone()
        return got

    here, plain = run(shift), run(0)
    for name in here:
        a, b = here[name].cpu().double(), plain[name].cpu().double()
        assert a.isfinite().all(), name
        # (both were rounded from values that float32 sums in another order made: two halves of a step of the larger, not one)
        bound = 2 * ro.HALF_STEP[dtype] * torch.maximum(a.abs(), b.abs()) + ro.ROUNDINGS * 2.0 ** -24 * (b.abs() + b.abs().mean() + 1)
        assert ((a - b).abs() <= bound).all(), name


def test_two_streams_at_once():
    """The same join on two streams and two threads: nothing is shared between calls."""
    import threading

    r = lib()
    x, f, w = torch.randn(3000, 1024, device=DEV), torch.randn(3000, 1024, device=DEV), torch.rand(1024, device=DEV)
    g = torch.randn(3000, 1024, device=DEV)
    state = r.dropout_state(5, DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, f, w)]
        h, y = r.residual_join(leaves[0], leaves[1], branch_norm="rms", branch_weight=leaves[2], dropout=0.2, state=state, next_norm="layer")
        return [h, y] + list(torch.autograd.grad([h, y], leaves, [g, g]))

    want = [t.detach().clone() for t in step()]
    torch.cuda.synchronize()
    got, streams = {}, [torch.cuda.Stream() for _ in range(2)]

    def work(k):
        with torch.cuda.stream(streams[k]):
            for _ in range(10):
                got[k] = [t.detach().clone() for t in step()]

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        for a, b in zip(got[k], want):
            assert torch.equal(a, b)


def test_gradients_of_expanded_inputs():
    r = lib()
    x = torch.randn(1, 5, 48, device=DEV, requires_grad=True)
    f, gate = torch.randn(4, 5, 48, device=DEV), torch.randn(1, device=DEV, requires_grad=True)
    h = r.residual_join(x.expand(4, 5, 48), f, gate=gate)
    dx, dg = torch.autograd.grad(h, [x, gate], torch.ones_like(h))
    assert torch.equal(dx, torch.full_like(dx, 4.0))
    ro.assert_near(dg, f.cpu().double().sum().reshape(1), f.cpu().double().abs().sum().reshape(1), "dgate")
