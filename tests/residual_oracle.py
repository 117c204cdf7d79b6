"""Plain 64-bit statements of the residual-stream operators, with the magnitudes that bound a float32 evaluation's rounding.

``join64`` returns {name: (value, magnitude)}.  A magnitude is the same formula with every term replaced by its absolute value (and by
a magnitude where the term is itself computed), so that a float32 evaluation of n roundings, each at most half a step of what it
rounds, is off by at most about n * 2^-24 times it.  A kernel's longest chain: two statistics of a row for each of two norms and two sums
over a row for each of their gradients, each of at most 8 * ceil(C / 2048) + 13 additions, and some 30 operations between them; sums over R
rows add at most R / 148 + 40 more.  ROUNDINGS covers rows to 8192 elements and the row counts used here.  An output's own rounding is half a
step of its type.
"""
import numpy as np
import torch

ROUNDINGS = 400
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}   # half a step of float16's subnormals


def philox(counter, key):
    """Philox4x32-10 of integer arrays; counter: four of 32 bits, key: two."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p):
    return int(np.floor(p * 2.0 ** 32 + 0.5))


def numbers(seed, offset, first, n):
    """The 32-bit numbers of the elements first .. first + n - 1."""
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    i = np.arange(first, first + n, dtype=np.uint64)
    block, digit = i >> np.uint64(3), (i & np.uint64(7)).astype(np.int64)

    def of(second):
        words = philox([block & np.uint64(0xFFFFFFFF), (block >> np.uint64(32)) | np.uint64(second << 31), np.full_like(block, offset & 0xFFFFFFFF),
                        np.full_like(block, offset >> 32)], (seed & 0xFFFFFFFF, seed >> 32))
        word = np.choose(digit >> 1, words)
        return np.where(digit & 1, word >> np.uint64(16), word & np.uint64(0xFFFF))

    return of(0) * np.uint64(65536) + of(1)


def keeps(p, seed, offset, n, first=0):
    return torch.from_numpy(numbers(seed, offset, first, n) >= np.uint64(threshold(p)))


def drop_scale(p):
    return 2.0 ** 32 / (2 ** 32 - threshold(p)) if threshold(p) < 2 ** 32 else 0.0


def _mean(t):
    return t.mean(dim=-1, keepdim=True)


def _norm(t, big, kind, eps):
    """normalised rows, their magnitude, mean and reciprocal deviation"""
    mean = _mean(t) if kind == "layer" else torch.zeros_like(t[..., :1])
    r = 1.0 / torch.sqrt(_mean((t - mean) ** 2) + eps)
    # (an error of t changes r by up to as much again)
    return (t - mean) * r, 2 * r * (big + _mean(big)) + (t - mean).abs() * r, mean, r


def join64(x, f, after, aw, ab, gate, skip, branch, kept, scale, before, bw, bb, eps, dh, dy):
    """x, f, dh, dy: 64-bit [rows..., C]; gate: broadcastable; kept: truth values or None.  f None: the norm alone."""
    one, zero = torch.ones((), dtype=torch.float64), torch.zeros((), dtype=torch.float64)
    aw, bw, ab, bb = (one if aw is None else aw), (one if bw is None else bw), (zero if ab is None else ab), (zero if bb is None else bb)
    out = {}
    h, hb = x, x.abs()
    if f is not None:
        t = f if kept is None else torch.where(kept, f * scale, 0.0)
        tb = t.abs()
        xh, xb = (t, tb) if after is None else _norm(t, tb, after, eps)[:2]
        r = None if after is None else _norm(t, tb, after, eps)[3]
        n, nb = xh * aw + ab, xb * aw.abs() + ab.abs()
        g = one if gate is None else gate
        h, hb = skip * x + branch * g * n, abs(skip) * x.abs() + abs(branch) * g.abs() * nb
        out["h"] = (h, hb)
    if before is not None:
        zh, zb, _, q = _norm(h, hb, before, eps)
        out["y"] = (zh * bw + bb, zb * bw.abs() + bb.abs())
    if dh is None and dy is None:
        return out
    d, db = (torch.zeros_like(x),) * 2 if dh is None else (dh, dh.abs())
    lead = tuple(range(x.dim() - 1))
    if dy is not None:
        u, ub = dy * bw, dy.abs() * bw.abs()
        layer = before == "layer"
        # (each part also carries what an error of q makes of it)
        d = d + q * (u - (_mean(u) if layer else 0.0) - zh * _mean(u * zh))
        db = db + 2 * q * (ub + (_mean(ub) if layer else 0.0) + zb * _mean(ub * zb))
        out["dbw"], out["dbb"] = ((dy * zh).sum(lead), (dy.abs() * zb).sum(lead)), (dy.sum(lead), dy.abs().sum(lead))
    if f is None:
        out["dx"] = (d, db)
        return out
    out["dx"] = (skip * d, abs(skip) * db)
    d, db = branch * d, abs(branch) * db
    if gate is not None:
        full, fb = d * n, db * nb
        shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
        dims = [k for k in range(x.dim()) if shape[k] == 1 and x.shape[k] != 1]
        out["dgate"] = tuple((v.sum(dims, keepdim=True) if dims else v).reshape(gate.shape) for v in (full, fb))
        d, db = d * gate, db * gate.abs()
    if after is not None:
        out["daw"], out["dab"] = ((d * xh).sum(lead), (db * xb).sum(lead)), (d.sum(lead), db.sum(lead))
        v, vb = d * aw, db * aw.abs()
        layer = after == "layer"
        d = r * (v - (_mean(v) if layer else 0.0) - xh * _mean(v * xh))
        db = 2 * r * (vb + (_mean(vb) if layer else 0.0) + xb * _mean(vb * xb))
    if kept is not None:
        d, db = torch.where(kept, d * scale, 0.0), db * scale
    out["df"] = (d, db)
    return out


def assert_near(got, want, magnitude, name):
    """got: a tensor of its type; within its rounding and ROUNDINGS float32 roundings of the 64-bit value."""
    g = got.detach().cpu().double()
    assert g.shape == want.shape, f"{name}: shape {tuple(g.shape)}, not {tuple(want.shape)}"
    bound = HALF_STEP[got.dtype] * want.abs() + SMALLEST[got.dtype] + ROUNDINGS * 2.0 ** -24 * magnitude * (1 + HALF_STEP[got.dtype])
    off = (g - want).abs()
    bad = ~(off <= bound)   # (NaN is bad)
    if bad.any():
        at = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {g.reshape(-1)[at]} not {want.reshape(-1)[at]} "
                             f"+- {bound.expand_as(want).reshape(-1)[at]}")
