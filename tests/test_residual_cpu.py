"""Residual-stream operators without a GPU: the generator's published vectors, the 64-bit statements against differences, refusals."""
import ctypes

import numpy as np
import pytest
import torch

import residual_oracle as ro


def test_generator_known_answers():
    """Known answers published with the generator (counter, key -> block)."""
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in ro.philox(counter, key)) == want


def test_shares_of_dropped_elements():
    """A million elements: the share of dropped ones is within five standard deviations of p."""
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        share = 1.0 - ro.keeps(p, 12345, 678, n).double().mean().item()
        assert abs(share - p) < 5 * (p * (1 - p) / n) ** 0.5


@pytest.mark.parametrize("after,before", [(None, "rms"), ("rms", None), ("layer", "rms"), ("rms", "layer"), (None, None)])
def test_formulas_against_differences(after, before):
    """Central differences in 64 bits: error about step^2 and 2^-53 / step, both under 1e-9 of values of order one at a step of 1e-5."""
    gen = torch.Generator().manual_seed(1)
    shape, C = (2, 3, 5), 5

    def normal(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)

    v = dict(x=normal(*shape), f=normal(*shape), gate=normal(2, 1, C))
    if after:
        v.update(aw=1 + 0.1 * normal(C), ab=normal(C))
    if before:
        v.update(bw=1 + 0.1 * normal(C), bb=normal(C))
    kept = torch.rand(shape, generator=gen) > 0.3
    dh, dy = normal(*shape), normal(*shape) if before else None

    def forward(v, grads):
        return ro.join64(v["x"], v["f"], after, v.get("aw"), v.get("ab"), v["gate"], 0.75, 0.5, kept, 1.25, before, v.get("bw"), v.get("bb"),
                         1e-3, dh if grads else None, dy if grads else None)

    def loss(v):
        o = forward(v, False)
        return float((o["h"][0] * dh).sum() + ((o["y"][0] * dy).sum() if before else 0.0))

    got, step = forward(v, True), 1e-5
    for name, value in v.items():
        want = torch.zeros_like(value).reshape(-1)
        for i in range(value.numel()):
            side = []
            for sign in (1, -1):
                moved = dict(v)
                moved[name] = value.clone()
                moved[name].view(-1)[i] += sign * step
                side.append(loss(moved))
            want[i] = (side[0] - side[1]) / (2 * step)
        assert torch.allclose(got["d" + name][0].reshape(-1), want, rtol=1e-7, atol=1e-7), name


def test_entry_points_refuse():
    """Argument errors come before any CUDA call: status < 0 and a message."""
    from spiky_b200 import _native as nat

    L = nat.lib()
    assert L.lutb_dropout(7, 8, 0.5, None, 0, None, None, None) == -3
    assert L.lutb_dropout(nat.F32, -1, 0.5, None, 0, None, None, None) == -2
    for p in (-0.1, 1.5, float("nan")):
        assert L.lutb_dropout(nat.F32, 8, p, None, 0, None, None, None) == -2
    assert L.lutb_dropout(nat.F32, 8, 0.5, None, 0, None, None, None) == -1
    assert L.lutb_dropout(nat.F32, 8, 0.5, 8, -1, 16, 16, None) == -2
    assert L.lutb_dropout(nat.F32, 8, 0.5, 8, 0, 18, 16, None) == -5
    assert L.lutb_dropout(nat.F32, 0, 0.5, None, 0, None, None, None) == 0
    assert L.lutb_dropout_advance(None, 1, None, None) == -1
    assert L.lutb_dropout_advance(8, -1, 8, None) == -2

    def cfg(**more):
        v = dict(rows=4, width=8, eps=1e-6, before=nat.NORM_RMS, skip_scale=1.0, branch_scale=1.0)
        v.update(more)
        return ctypes.byref(nat.JoinCfg(**v))

    def forward(c, x=16, f=16, gate=None, aw=None, random=None, h=16, y=16, stats=None):
        return L.lutb_join_forward(c, x, f, gate, aw, None, None, None, random, h, y, stats, None)

    assert L.lutb_join_forward(None, *[None] * 12) == -1
    assert forward(cfg(rows=0)) == 0
    for bad in (dict(width=0), dict(width=2 ** 31), dict(rows=-1), dict(rows=2 ** 62), dict(gate_rows=3), dict(gate_rows=-1), dict(eps=0.0), dict(eps=float("nan")),
                dict(skip_scale=float("inf")), dict(dropout=2.0), dict(dropout=float("nan")), dict(site=-1)):
        assert forward(cfg(**bad)) == -2, bad
    for bad in (dict(stream_type=3), dict(stream_type=nat.BF16), dict(stream_type=nat.BF16, branch_type=nat.F16), dict(param_type=nat.F16),
                dict(gate_type=nat.BF16), dict(after=3), dict(before=-1)):
        assert forward(cfg(**bad)) == -3, bad
    for bad in (dict(x=None), dict(f=None), dict(h=None), dict(y=None), dict(gate=16)):
        assert forward(cfg(), **bad) == -1, bad
    assert forward(cfg(gate_rows=4)) == -1 and forward(cfg(dropout=0.5)) == -1 and forward(cfg(before=nat.NORM_NONE)) == -1
    assert forward(cfg(), x=18) == -5 and forward(cfg(), stats=8) == -5 and forward(cfg(dropout=0.5), random=4) == -5

    def backward(c, x=16, f=16, gate=None, stats=16, dh=16, dy=16, dgate=None, daw=None, dbw=None, ws=None, size=0):
        return L.lutb_join_backward(c, x, f, gate, None, None, None, None, stats, dh, dy, None, None, dgate, daw, None, dbw, None, ws, size, None)

    for bad in (dict(x=None), dict(stats=None), dict(dh=None, dy=None), dict(dgate=16), dict(f=None), dict(dy=None, dbw=16)):
        assert backward(cfg(), **bad) == -1, bad
    assert backward(cfg(), daw=16) == -3 and backward(cfg(before=nat.NORM_NONE)) == -3
    assert backward(cfg(), dbw=16) == -4 and backward(cfg(), dbw=16, ws=16, size=8) == -4
    assert L.lutb_join_backward_workspace(cfg()) > 0 and L.lutb_join_backward_workspace(cfg(width=0)) == 0


def test_python_refuses_cpu_tensors():
    from spiky_b200 import residual as r

    x, state = torch.zeros(2, 8), r.dropout_state(1, "cpu")
    for call in (lambda: r.counter_dropout(x, 0.5, state), lambda: r.row_norm(x), lambda: r.residual_join(x, x),
                 lambda: r.take_dropout_state(state, 1), lambda: r.counter_dropout([1.0], 0.5, state), lambda: r.residual_join(x, None)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        r.CounterDropout(1.5)
    with pytest.raises(ValueError):
        r.RowNorm(8, kind="batch")
    with pytest.raises(ValueError):
        r.ResidualJoin(8, dropout=-0.1)


def test_state_wraps_to_64_bits():
    from spiky_b200 import residual as r

    s = r.dropout_state(2 ** 64 - 1, "cpu", offset=2 ** 63)
    assert s.tolist() == [-1, -2 ** 63]
    assert np.array_equal(ro.numbers(-1, 5, 0, 16), ro.numbers(2 ** 64 - 1, 5, 0, 16))


def test_gate_rows():
    from spiky_b200.residual import _gate_rows

    x = torch.zeros(2, 3, 4, 5)
    for shape, rows in (((5,), 24), ((1, 5), 24), ((2, 1, 1, 5), 12), ((2, 3, 1, 5), 4), ((2, 3, 4, 5), 1)):
        assert _gate_rows(torch.zeros(shape), x) == rows
    for shape in ((), (4,), (2, 1, 4, 5), (3, 4, 5), (1, 2, 3, 4, 5), (3, 1, 1, 5)):
        with pytest.raises(ValueError):
            _gate_rows(torch.zeros(shape), x)
