"""What joins blocks in a residual stream: dropout without a stored mask, norms of rows, and the join of a block's output.

No counterpart in the reference, whose transformer composes torch's dropout, ``BatchNorm1d`` and a sum
(src/spiky/lut/LUTTransformer.py:69-271).  Here each is one kernel and one pass over the data, forward and backward:

* ``counter_dropout(x, p, state, site)``: the mask is a function of the seed, an offset and the element's number, formed again in
  the backward pass; nothing of the size of ``x`` is kept.
* ``row_norm(x, weight, bias, kind)``: RMS or layer norm over the last dimension, the norm before a block.
* ``residual_join(x, branch, ...)``: ``h = skip_scale * x + branch_scale * gate * N(drop(branch))``, with the norm ``N`` after the
  block, and in the same pass ``y = N'(h)``, the norm before the next block.  Only what the gradients need is kept: nothing of the
  size of ``x`` where there is no norm and no learned gate.

float32, bfloat16 and float16; a float32 stream may carry a 16-bit branch.  Sums, norms and their statistics are float32, every
output is rounded once.  ``CounterDropout``, ``RowNorm`` and ``ResidualJoin`` are the modules; ``LUTTransformer`` uses them.  Ordinary calls run through
the native host side (host/residual_calls.cpp); the functions here define them all and take the rest.

Argument mistakes raise ``ValueError``, mistakes of type or device ``RuntimeError``; there is no CPU path.  Traces, forward-mode
derivatives and second derivatives of joins raise too: none is left out in silence.  Tensors that are not contiguous are copied.
Work goes to torch's current stream of the tensors' device.
"""
import ctypes
import math
import sys
import warnings

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn

from . import _native
from ._native import JoinCfg

_calls = None   # the native host side (host/residual_calls.cpp), once a call has asked for it


class _PythonRoute:
    """What stands in for the native host side where there is none: leaves every call to the functions below."""

    @staticmethod
    def join(*args):
        return None

    dropout = take = join


def _native_calls():
    global _calls
    try:
        _calls = _native.residual_calls()
    except (ImportError, RuntimeError) as e:
        warnings.warn(f"residual operators take the Python route, at about twice the host time: {e}", RuntimeWarning, stacklevel=4)
        _calls = _PythonRoute
    return _calls


_TYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
_NORMS = {None: _native.NORM_NONE, "rms": _native.NORM_RMS, "layer": _native.NORM_LAYER}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)   # (a stream's object has no such number under torch.compile)


def _refuse_recording():
    """The kernels are called past torch: a trace or a graph of torch's operators would keep the outputs' allocation alone, and the sizes of
    this call whatever it is given later."""
    fx = sys.modules.get("torch.fx.experimental.proxy_tensor")
    if torch.jit.is_tracing() or (fx is not None and fx.get_proxy_mode() is not None):
        raise RuntimeError("residual operators cannot be traced: their kernels would be missing from what is recorded")


def _check_data(t, name, device=None):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be on CUDA: spiky_b200 has no CPU path")
    if t.layout != torch.strided:
        raise RuntimeError(f"{name} must be a dense tensor")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on {device}")


def _check_tangent(t, name):
    if t is not None and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} has a tangent: residual operators have no forward-mode derivatives")


def _check_dropout(p, state, site, device):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
    if not 0 <= site < 2 ** 63:
        raise ValueError("site must be a number from 0 to 2**63 - 1")
    if p == 0.0:
        return
    if not isinstance(state, torch.Tensor) or state.dtype != torch.int64 or state.shape != (2,) or not state.is_contiguous():
        raise RuntimeError("state must be a contiguous int64 tensor of two elements (dropout_state)")
    if state.device != device:
        raise RuntimeError(f"state must be on {device}")


# ------------------------------------------------------------------------------------------------ dropout
def dropout_state(seed, device, offset=0):
    """int64 [2] on ``device``: the seed (any 64 bits) and the offset that a dropout reads when its kernel runs."""
    wrap = [(int(v) + 2 ** 63) % 2 ** 64 - 2 ** 63 for v in (seed, offset)]
    return torch.tensor(wrap, dtype=torch.int64, device=device)


def drawn_seed():
    """A seed from torch's generator of the host."""
    return int(torch.randint(2 ** 62, (1,), device="cpu"))


def replica_site(replica=None):
    """The first site of a replica's dropouts: ``site = replica_site() + k`` gives data-parallel replicas masks of their own from one state.
    ``replica``: a number below 2**15, by default the process's rank in torch.distributed's default group, 0 without one.

    The state is a buffer, and buffers are made alike on all ranks (``broadcast_structure``, ``DistributedDataParallel``, a checkpoint that
    all load): what tells replicas apart must not lie in it.  Replicas are 2**48 sites apart, more than any run's dropouts.
    """
    if replica is None:
        dist = torch.distributed
        replica = dist.get_rank() if dist.is_available() and dist.is_initialized() else 0
    if not 0 <= replica < 2 ** 15:
        raise ValueError("replica must be a number from 0 to 2**15 - 1")
    return int(replica) << 48


def take_dropout_state(state, count):
    """A copy of ``state`` for ``count`` dropouts (their sites 0 .. count - 1); the offset in ``state`` moves on by ``count``.

    A part that ``torch.utils.checkpoint`` runs again in the backward pass has to be handed its copy from outside: one taken inside would be
    another one the second time, with another mask.  Taking one during a backward pass is therefore an error.
    """
    if torch._C._current_graph_task_id() != -1:
        raise RuntimeError("a dropout state is taken during a backward pass: take it outside the part that is run again (torch.utils.checkpoint) "
                           "and hand it in, or the mask would be another one than the outputs were made with")
    used = (_calls or _native_calls()).take(state, count)
    if used is not None:
        return used
    _refuse_recording()
    _check_dropout(1.0, state, 0, state.device if isinstance(state, torch.Tensor) else None)
    if not state.is_cuda:
        raise RuntimeError("state must be on CUDA: spiky_b200 has no CPU path")
    if count < 0:
        raise ValueError("count < 0")
    used = torch.empty_like(state)
    with torch.cuda.device(state.device):
        _native.check(_native.lib().lutb_dropout_advance(_ptr(state), int(count), _ptr(used), _stream(state.device)))
    torch.autograd.graph.increment_version(state)
    return used


def _whole(t):
    """As the kernels read it: contiguous, no lazy negation."""
    return None if t is None else t.detach().resolve_neg().contiguous()


def _expect(t, like, numel, name):
    """What a backward pass is handed can come from hooks: the kernels get nothing that is not what the forward pass had."""
    dtype, device = like
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or t.numel() != numel or t.layout != torch.strided:
        raise RuntimeError(f"{name} is not what the forward pass saved: {numel} elements of {dtype} on {device}")
    _check_tangent(t, name)
    return _whole(t)


def _dropout(x, p, state, site):
    x = _whole(x)
    y = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _native.check(_native.lib().lutb_dropout(_TYPES[x.dtype], x.numel(), p, _ptr(state), site, _ptr(x), _ptr(y), _stream(x.device)))
    return y


class _CounterDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, state, site):
        ctx.p, ctx.site = p, site
        ctx.save_for_backward(state)
        return _dropout(x, p, state, site)

    @staticmethod
    def backward(ctx, dy):
        state, = ctx.saved_tensors
        _expect(state, (torch.int64, dy.device), 2, "state")
        return counter_dropout(dy, ctx.p, state, ctx.site), None, None, None


def counter_dropout(x, p, state, site=0):
    """Inverted dropout of ``x`` whose mask follows from ``state`` (``dropout_state``) and ``site`` alone.

    Element ``i`` (row by row) is dropped when a 32-bit number of the Philox4x32-10 generator with the key ``seed`` and the counter
    ``(i // 8, offset + site)`` is below ``round(p * 2**32)``; what stays is scaled by the reciprocal of the rest's share, what is
    dropped is 0 even where ``x`` is infinite or NaN.  The backward pass reads ``state`` again: leave it as it was until then
    (``take_dropout_state`` hands out copies).
    """
    y = (_calls or _native_calls()).dropout(x, p, state, site)
    if y is not None:
        return y
    p, site = float(p), int(site)
    _check_data(x, "x")
    _check_dropout(p, state, site, x.device)
    if p == 0.0:
        return x.clone()
    _refuse_recording()
    _check_tangent(x, "x")
    if x.requires_grad and torch.is_grad_enabled():
        return _CounterDropout.apply(x, p, state, site)
    return _dropout(x, p, state, site)


# ------------------------------------------------------------------------------------------------ joins and norms
def _check_vector(t, name, width, branch_type, device):
    _check_data(t, name, device)
    if t.shape != (width,):
        raise ValueError(f"{name} must have shape ({width},), got {tuple(t.shape)}")
    if t.dtype not in (torch.float32, branch_type):
        raise RuntimeError(f"{name} must be float32 or of the branch's type")


def _gate_rows(gate, x):
    """How many rows of x share a row of the gate; ValueError where its shape says something else."""
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    if gate.dim() == 0 or len(shape) > x.dim() or shape[-1] != x.shape[-1]:
        raise ValueError(f"a gate for {tuple(x.shape)} has one element or rows of {x.shape[-1]}, got {tuple(gate.shape)}")
    lead, mine = x.shape[:-1], shape[:-1]
    k = len(lead)
    while k > 0 and mine[k - 1] == 1:
        k -= 1
    if tuple(mine[:k]) != tuple(lead[:k]):
        raise ValueError(f"a gate for {tuple(x.shape)} is shared by trailing dimensions only, got {tuple(gate.shape)}")
    return math.prod(lead[k:])


# Which saved tensors (of _Join.backward's names) the gradients of (x, branch, gate, branch_weight, branch_bias, next_weight, next_bias)
# depend on, where the next norm has no gradient to hand on and where it has one; of the first, those in brackets with a norm of the branch alone.
_SOURCES = (((), ()), ((2,), (1, 3)), ((1,), (3, 4)), ((1, 2), ()), ((2,), ()), ((), ()), ((), ()))


def _sources(cfg, k, dy):
    if dy is not None:
        return range(6 if k < 6 else 0)
    return _SOURCES[k][0] + (_SOURCES[k][1] if cfg.after != _native.NORM_NONE else ())


class _Once(torch.autograd.Function):
    """A gradient tied to what it was formed from, so that a second derivative raises instead of being left out."""

    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.detach()

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("a residual join is differentiable once")


class _Join(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, branch, gate, aw, ab, bw, bb, state, stats):
        h, y = _join_forward(cfg, x, branch, gate, aw, ab, bw, bb, state, stats)
        ctx.cfg = cfg
        given = (x, branch, gate, aw, ab, bw, bb)
        ctx.had = [None if t is None else (t.shape, t.dtype, t.device) for t in given]
        ctx.of_grads = [None if t is None else (t.dtype, t.device) for t in (h, y)]
        # what the backward pass reads: the stream for the next norm, the branch for norms and the gate's gradient
        norms = cfg.after != _native.NORM_NONE or cfg.before != _native.NORM_NONE
        kept = [x if cfg.before != _native.NORM_NONE else None, branch if norms or ctx.needs_input_grad[3] else None, gate, aw, ab, bw,
                state, stats]
        ctx.kept = [None if t is None else ((t.dtype, t.device), t.numel()) for t in kept]
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*kept)
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        if dh is None and dy is None:
            return (None,) * 10
        _refuse_recording()
        saved = ctx.saved_tensors   # (once: hooks may run a part again for it)
        with torch.no_grad():
            grads = _Join.gradients(ctx, saved, dh, dy)
        if torch.is_grad_enabled():   # a graph is asked for: one that says so when it is used
            for k, grad in enumerate(grads):
                of = [t for t in (dh, dy) + tuple(saved[i] for i in _sources(ctx.cfg, k, dy)) if t is not None and t.requires_grad]
                if grad is not None and of:
                    grads[k] = _Once.apply(grad, *of)
        return (None, *grads, None, None)

    @staticmethod
    def gradients(ctx, saved, dh, dy):
        cfg, need = ctx.cfg, ctx.needs_input_grad
        names = ("x", "branch", "gate", "branch_weight", "branch_bias", "next_weight", "state", "stats")
        con = [None if kept is None else _expect(t, *kept, name) for t, kept, name in zip(saved, ctx.kept, names)]
        shape, _, device = ctx.had[0]
        dh, dy = (None if t is None else _expect(t, like, shape.numel(), "the gradient") for t, like in zip((dh, dy), ctx.of_grads))

        def like(k, wanted=True):
            had = ctx.had[k]
            return torch.empty(had[0], dtype=had[1], device=had[2]) if had is not None and need[k + 1] and wanted else None

        dx, df, dgate, daw, dab = (like(k) for k in range(5))
        dbw, dbb = like(5, dy is not None), like(6, dy is not None)
        with torch.cuda.device(device):
            L = _native.lib()
            ws, size = None, 0
            if any(t is not None for t in (daw, dab, dbw, dbb)) or (dgate is not None and cfg.gate_rows > 1):
                size = L.lutb_join_backward_workspace(ctypes.byref(cfg))
                ws = torch.empty(size, dtype=torch.uint8, device=device)
            _native.check(L.lutb_join_backward(
                ctypes.byref(cfg), *(_ptr(t) for t in con), _ptr(dh), _ptr(dy), _ptr(dx), _ptr(df),
                _ptr(dgate), _ptr(daw), _ptr(dab), _ptr(dbw), _ptr(dbb), _ptr(ws), size, _stream(device)))
        return [dx, df, dgate, daw, dab, dbw, dbb]


def _join_forward(cfg, x, branch, gate, aw, ab, bw, bb, state, stats):
    con = [_whole(t) for t in (x, branch, gate, aw, ab, bw, bb)]
    branch_type = [k for k, v in _TYPES.items() if v == cfg.branch_type][0]
    h = None if branch is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y = torch.empty(x.shape, dtype=branch_type, device=x.device) if cfg.before != _native.NORM_NONE else None
    with torch.cuda.device(x.device):
        _native.check(_native.lib().lutb_join_forward(ctypes.byref(cfg), *(_ptr(t) for t in con), _ptr(state), _ptr(h), _ptr(y), _ptr(stats),
                                                      _stream(x.device)))
    return h, y


def _join(x, branch, branch_type, after, aw, ab, gate, skip_scale, branch_scale, p, state, site, before, bw, bb, eps):
    _refuse_recording()
    _check_data(x, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("x must have rows of at least one element")
    width, device = x.shape[-1], x.device
    if after not in _NORMS or before not in _NORMS:
        raise ValueError("a norm is None, 'rms' or 'layer'")
    if branch is not None:
        _check_data(branch, "branch", device)
        if branch.shape != x.shape:
            raise ValueError(f"branch must have the shape of x, {tuple(x.shape)}, got {tuple(branch.shape)}")
    if branch_type not in _TYPES or (x.dtype != branch_type and x.dtype != torch.float32):
        raise RuntimeError("the branch must have the type of x, or x must be float32")
    for kind, w, b, name in ((after, aw, ab, "branch"), (before, bw, bb, "next")):
        if kind is None and (w is not None or b is not None):
            raise ValueError(f"{name}_weight and {name}_bias need {name}_norm")
    params = [(t, n) for t, n in ((aw, "branch_weight"), (ab, "branch_bias"), (bw, "next_weight"), (bb, "next_bias")) if t is not None]
    for t, n in params:
        _check_vector(t, n, width, branch_type, device)
        if t.dtype != params[0][0].dtype:
            raise RuntimeError("weights and biases must have one type")
    p, site = float(p), int(site)
    skip_scale, branch_scale, eps = float(skip_scale), float(branch_scale), float(eps)
    _check_dropout(p, state, site, device)
    if not (math.isfinite(skip_scale) and math.isfinite(branch_scale)):
        raise ValueError("scales must be finite")
    if not (math.isfinite(eps) and ctypes.c_float(eps).value > 0.0):
        raise ValueError("eps must be positive")
    gate_rows = 0
    if gate is not None:
        _check_data(gate, "gate", device)
        if gate.dtype not in (torch.float32, branch_type):
            raise RuntimeError("gate must be float32 or of the branch's type")
        if gate.numel() == 1:   # (a learned scalar: autograd sums the row of its gradient, in float32 up to the one rounding behind the cast)
            gate = gate.float().reshape(1).expand(width)
        gate_rows = _gate_rows(gate, x)
    rows = x.numel() // width
    cfg = JoinCfg(rows=rows, width=width, gate_rows=gate_rows if rows else 0, site=site, dropout=p, stream_type=_TYPES[x.dtype],
                  branch_type=_TYPES[branch_type], param_type=_TYPES[params[0][0].dtype if params else torch.float32],
                  gate_type=_TYPES[gate.dtype if gate is not None else torch.float32], after=_NORMS[after], before=_NORMS[before], eps=eps,
                  skip_scale=skip_scale, branch_scale=branch_scale, reserved0=0)
    state = state if p > 0.0 else None
    tensors = (x, branch, gate, aw, ab, bw, bb)
    for t, name in zip(tensors, ("x", "branch", "gate", "branch_weight", "branch_bias", "next_weight", "next_bias")):
        _check_tangent(t, name)
    if rows == 0 and gate is not None:   # no gate row is read; its gradient is nothing, or zeros
        branch, gate = branch * gate.to(branch.dtype), None
        tensors = (x, branch, gate, aw, ab, bw, bb)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        stats = torch.empty((rows, 4), dtype=torch.float32, device=device) if after is not None or before is not None else None
        return _Join.apply(cfg, *tensors, state, stats)
    return _join_forward(cfg, *tensors, state, None)


def row_norm(x, weight=None, bias=None, kind="rms", eps=1e-6, dtype=None):
    """``N(x) * weight + bias`` over the last dimension: ``kind`` 'rms' is ``x / sqrt(mean(x^2) + eps)``, 'layer' is
    ``(x - mean) / sqrt(mean((x - mean)^2) + eps)``.  ``dtype``: the result's, that of ``x`` or a 16-bit type of a float32 ``x``."""
    got = (_calls or _native_calls()).join(x, None, dtype, None, None, None, None, 1.0, 1.0, 0.0, None, 0, kind, weight, bias, eps)
    if got is not None:
        return got[1]
    if kind is None:
        raise ValueError("kind is 'rms' or 'layer'")
    _check_data(x, "x")
    return _join(x, None, x.dtype if dtype is None else dtype, None, None, None, None, 1.0, 1.0, 0.0, None, 0, kind, weight, bias, eps)[1]


def residual_join(x, branch, *, branch_norm=None, branch_weight=None, branch_bias=None, gate=None, skip_scale=1.0, branch_scale=1.0,
                  dropout=0.0, state=None, site=0, next_norm=None, next_weight=None, next_bias=None, eps=1e-6):
    """``h = skip_scale * x + branch_scale * gate * N(drop(branch))``, and with ``next_norm`` also ``y = N'(h)``: returns ``h`` or
    ``(h, y)``.

    ``x`` and ``branch`` have one shape, ``branch`` the type of ``x`` or a 16-bit one beside a float32 ``x``; ``h`` has the type of
    ``x``, ``y`` that of ``branch``.  ``branch_norm`` / ``next_norm``: None, 'rms' or 'layer' (see ``row_norm``), each with an optional
    weight and bias of the last dimension's size.  ``gate``: one element, a row for all (``[C]``), a row for each sequence
    (``[B, 1, C]``) or for each token, shared by trailing dimensions; float32 or the branch's type.  ``dropout``, ``state`` and
    ``site``: as ``counter_dropout`` of the branch.  ``y`` is formed from ``h`` before its rounding.
    """
    if branch is None:
        raise RuntimeError("branch must be a tensor")
    got = (_calls or _native_calls()).join(x, branch, None, branch_norm, branch_weight, branch_bias, gate, skip_scale, branch_scale, dropout, state,
                                           site, next_norm, next_weight, next_bias, eps)
    if got is not None:
        return got[0] if next_norm is None else got
    _check_data(branch, "branch")
    h, y = _join(x, branch, branch.dtype, branch_norm, branch_weight, branch_bias, gate, skip_scale, branch_scale, dropout, state, site,
                 next_norm, next_weight, next_bias, eps)
    return h if next_norm is None else (h, y)


# ------------------------------------------------------------------------------------------------ modules
class CounterDropout(nn.Module):
    """``nn.Dropout`` with a mask that is never stored.  ``state`` is a buffer: checkpoints carry it on, replayed graphs move it on.  ``seed``: by
    default drawn from torch's generator, so that two modules have different masks.  ``replica``: see ``replica_site``; by default each rank of a
    data-parallel model has masks of its own, with one seed and one state.

    A part that ``torch.utils.checkpoint`` runs again gets its state from outside: ``checkpoint(part, x, drop.take_state())`` with
    ``drop(x, state)`` in it; without one the run in the backward pass raises.
    """

    replica = None   # (of modules that were pickled before it)

    def __init__(self, p=0.5, seed=None, device=None, replica=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
        if replica is not None:
            replica_site(replica)   # (refuses)
        self.p, self.replica = float(p), replica
        self.register_buffer("state", dropout_state(drawn_seed() if seed is None else seed, device))

    def take_state(self):
        """The state of one call, which moves on; for ``forward``."""
        return take_dropout_state(self.state, 1)

    def forward(self, x, state=None):
        if not self.training or self.p == 0.0:
            return x
        return counter_dropout(x, self.p, self.take_state() if state is None else state, replica_site(self.replica))

    def extra_repr(self):
        return f"p={self.p}"


def _norm_parameters(module, name, kind, width, bias, device, dtype):
    if kind not in _NORMS:
        raise ValueError("a norm is None, 'rms' or 'layer'")
    weight = shift = None
    if kind is not None:
        weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        shift = nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None
    module.register_parameter(name + "weight", weight)
    module.register_parameter(name + "bias", shift)


class RowNorm(nn.Module):
    """``row_norm`` with its weight and, by default for 'layer', its bias."""

    def __init__(self, width, kind="rms", bias=None, eps=1e-6, device=None, dtype=None):
        super().__init__()
        if kind is None:
            raise ValueError("kind is 'rms' or 'layer'")
        self.width, self.kind, self.eps = width, kind, eps
        _norm_parameters(self, "", kind, width, kind == "layer" if bias is None else bias, device, dtype)

    def forward(self, x, dtype=None):
        return row_norm(x, self.weight, self.bias, self.kind, self.eps, dtype)

    def extra_repr(self):
        return f"{self.width}, kind={self.kind!r}, eps={self.eps}"


class ResidualJoin(nn.Module):
    """``residual_join`` with its parameters: the norms' weights (and, by default for 'layer', biases) and a gate row.

    ``forward(x, branch, state, site)`` returns ``(h, y)``, ``y`` is ``h`` without ``next_norm``.  Dropout needs a ``state``
    (``take_dropout_state``) and, in a data-parallel model, sites from ``replica_site`` on; it is off in evaluation mode.
    """

    def __init__(self, width, branch_norm=None, next_norm=None, gated=False, gate_init=1.0, skip_scale=1.0, branch_scale=1.0, dropout=0.0,
                 bias=None, eps=1e-6, device=None, dtype=None):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout probability has to be between 0 and 1, but got {dropout}")
        self.width, self.branch_norm, self.next_norm, self.eps = width, branch_norm, next_norm, eps
        self.skip_scale, self.branch_scale, self.dropout = float(skip_scale), float(branch_scale), float(dropout)
        for name, kind in (("branch_", branch_norm), ("next_", next_norm)):
            _norm_parameters(self, name, kind, width, kind == "layer" if bias is None else bias, device, dtype)
        self.gate = nn.Parameter(torch.full((width,), float(gate_init), device=device, dtype=dtype)) if gated else None

    def forward(self, x, branch, state=None, site=0):
        got = residual_join(x, branch, branch_norm=self.branch_norm, branch_weight=self.branch_weight, branch_bias=self.branch_bias,
                            gate=self.gate, skip_scale=self.skip_scale, branch_scale=self.branch_scale,
                            dropout=self.dropout if self.training else 0.0, state=state, site=site, next_norm=self.next_norm,
                            next_weight=self.next_weight, next_bias=self.next_bias, eps=self.eps)
        return (got, got) if self.next_norm is None else got

    def extra_repr(self):
        return (f"{self.width}, branch_norm={self.branch_norm!r}, next_norm={self.next_norm!r}, gated={self.gate is not None}, "
                f"dropout={self.dropout}")
