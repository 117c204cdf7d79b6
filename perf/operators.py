"""The residual-stream operators of ``spiky_b200.residual`` and their plain forms, as cases with inputs, outputs and work.

dropout  ``counter_dropout``: inverted dropout whose mask is a function of (seed, offset, element) and is never stored
norm     ``row_norm``: RMS or layer norm of every token, the norm before a block
join     ``residual_join``: a block's output through dropout, the norm after the block, gate and scale into the residual
         stream, and the norm before the next block

Where ``own`` is false the operators run in their plain form: elementary torch operations in 32 bits, rounded once at the end,
gradients by autograd.  A case with ``train`` is a forward and a backward pass and returns the gradients too.

The generator is Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011).  The tensor's
elements are numbered row by row; element ``i`` takes 16-bit digit ``i % 8`` of the block with the counter (i / 8, offset + site) and
the key ``seed``, and a second digit from the counter whose top bit of the first half is set.  It is dropped when the 32-bit number
that the two digits make is below round(p * 2^32).
"""
import math

import torch

own = False

DEVICE = "cuda"
LOW32 = 0xFFFFFFFF


def _case(name, op, sequences, length, width, stream, branch, train, **more):
    case = dict(op=op, sequences=sequences, length=length, width=width, stream=stream, branch=branch, train=train, params="float32",
                p=0.0, after="none", before="none", bias=False, gate="none", skip_scale=1.0, branch_scale=1.0, site=0)
    case.update(more)
    return dict(name=name, **case)


def listed():
    return [
        # the activations of a small character model's batch: 64 sequences of 128 tokens
        _case("dropout, character model", "dropout", 64, 128, 256, "float32", "float32", True, p=0.1, site=3),
        # a long batch in half precision, the stream of a wide model
        _case("dropout, large bf16", "dropout", 8, 2048, 4096, "bfloat16", "bfloat16", True, p=0.1, site=1),
        # a ragged batch: rows that end on no boundary
        _case("dropout, odd fp16", "dropout", 37, 101, 1001, "float16", "float16", True, p=0.25),
        # serving: one token's norm before a block
        _case("norm, one token", "norm", 1, 1, 4096, "bfloat16", "bfloat16", False, before="rms", params="bfloat16"),
        # the character model's norms, trained
        _case("norm, character model", "norm", 64, 128, 256, "float32", "float32", True, before="layer", bias=True),
        # the attention layer's stream of 32 long sequences; fp32 stream, bf16 block
        _case("norm, long sequences", "norm", 32, 1024, 1024, "float32", "bfloat16", True, before="rms"),
        # serving: one token between two blocks
        _case("join, one token", "join", 1, 1, 4096, "bfloat16", "bfloat16", False, after="rms", before="rms", branch_scale=0.5),
        # serving: a batch of tokens of requests, fp32 stream, bf16 block
        _case("join, token batch", "join", 96, 1, 2048, "float32", "bfloat16", False, after="none", before="layer", bias=True,
              gate="width"),
        # one block of the character model, trained with dropout
        _case("join, character model", "join", 64, 128, 256, "float32", "float32", True, p=0.1, before="layer", bias=True,
              branch_scale=0.5, site=2),
        # the long-sequence attention block: norms on both sides, a learned gate, dropout
        _case("join, long sequences", "join", 32, 1024, 1024, "float32", "float32", True, p=0.1, after="rms", before="rms",
              gate="width", site=5),
        # the largest: a wide stream in half precision, one gate row a sequence, layer norms with bias on both sides
        _case("join, wide bf16", "join", 8, 1536, 8192, "bfloat16", "bfloat16", True, p=0.05, after="layer", before="layer", bias=True,
              gate="sequence", skip_scale=0.875, site=7),
        # odd sizes: a ragged batch, width without a factor of two, a gate for each element
        _case("join, odd fp16", "join", 3, 1333, 1005, "float16", "float16", True, p=0.2, after="layer", before="rms",
              gate="element", site=1),
    ]


def draw(rng):
    op = rng.choice(["dropout", "norm", "join", "join"])
    stream, branch = rng.choice([("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "bfloat16"),
                                 ("float32", "float16")])
    train = rng.random() < 0.7
    width = int(round(16 * 2 ** rng.uniform(0, 9)))
    if rng.random() < 0.5:
        width = max(16, width // 64 * 64)
    most = 48 * 2 ** 20 // width
    tokens = int(math.exp(rng.uniform(0, math.log(most))))
    sequences = max(1, int(math.exp(rng.uniform(0, math.log(max(2, min(tokens, 256)))))))
    length = max(1, tokens // sequences)
    if op == "dropout":
        return dict(_case("", op, sequences, length, width, branch, branch, train, p=rng.choice([0.05, 0.1, 0.3, 0.5]),
                          site=rng.randrange(64)))
    after = rng.choice(["none", "rms", "layer"]) if op == "join" else "none"
    before = rng.choice(["rms", "layer"] + (["none"] if op == "join" else []))
    case = _case("", op, sequences, length, width, stream, branch, train, after=after, before=before,
                 bias=(after != "none" or before != "none") and rng.random() < 0.5, params=rng.choice(["float32", branch]))
    if op == "join":
        case.update(p=rng.choice([0.0, 0.1, 0.3]) if train else 0.0, gate=rng.choice(["none", "width", "sequence", "element"]),
                    skip_scale=rng.choice([1.0, 1.0, 0.875]), branch_scale=rng.choice([1.0, 0.5, 0.25]), site=rng.randrange(64))
    del case["name"]
    return case


def _type(name):
    return getattr(torch, name)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    shape = (case["sequences"], case["length"], case["width"])
    stream, branch, params = _type(case["stream"]), _type(case["branch"]), _type(case["params"])
    width = case["width"]

    def normal(size, scale=1.0, mean=0.0):
        return mean + scale * torch.randn(size, device=DEVICE, generator=gen)

    state = dict(case=case, leaves=[], ups=[])

    def leaf(name, value, dtype):
        value = value.to(dtype).requires_grad_(case["train"])
        state[name] = value
        if case["train"]:
            state["leaves"].append(name)

    def up(name, dtype):
        if case["train"]:
            state["ups"].append(name)
            state["d" + name] = normal(shape).to(dtype)

    # channels of a trained stream differ in size and are not centred
    size, centre = 0.5 + torch.rand(width, device=DEVICE, generator=gen), normal(width, 0.2)
    leaf("x", normal(shape) * size + centre, stream)
    if case["op"] == "join":
        leaf("f", 0.5 * normal(shape) * size + 0.5 * centre, branch)
    if case["gate"] != "none":
        gate = {"width": (width,), "sequence": (case["sequences"], 1, width), "element": shape}[case["gate"]]
        leaf("gate", normal(gate, 0.3, 0.7), branch if case["gate"] == "element" else params)
    for part in ("after", "before"):
        if case[part] != "none":
            leaf(part + "_weight", normal(width, 0.1, 1.0), params)
            if case["bias"]:
                leaf(part + "_bias", normal(width, 0.1), params)
    if case["op"] == "join":
        up("h", stream)
    if case["before"] != "none":
        up("y", branch)
    if case["op"] == "dropout":
        up("y", stream)
    if case["p"]:
        state["random"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), device=DEVICE, generator=gen).repeat(2)
        state["random"][1] = torch.randint(0, 2 ** 40, (1,), device=DEVICE, generator=gen)[0]
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _blocks(random, site, n, second):
    """The four 32-bit words of the generator's blocks 0 .. n-1, as int64 [n, 4]."""
    at, key0, key1, offset = torch.arange(n, device=random.device), random[0] & LOW32, random[0] >> 32 & LOW32, random[1] + site
    c0, c1, c2, c3 = at & LOW32, at >> 32 | second << 31, (offset & LOW32).expand(n), (offset >> 32 & LOW32).expand(n)
    for _ in range(10):   # the generator's ten rounds; products wrap in 64 bits, which leaves their words as they are
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & LOW32) ^ c1 ^ key0, p1 & LOW32, (p0 >> 32 & LOW32) ^ c3 ^ key1, p0 & LOW32
        key0, key1 = key0 + 0x9E3779B9 & LOW32, key1 + 0xBB67AE85 & LOW32
    return torch.stack([c0, c1, c2, c3], dim=1)


def _drop(x, p, random, site):
    """fp32 dropout of x."""
    n, below = x.numel(), int(math.floor(p * 2.0 ** 32 + 0.5))
    first, second = (torch.stack([w & 0xFFFF, w >> 16], dim=2).reshape(-1)[:n]
                     for w in (_blocks(random, site, (n + 7) // 8, k) for k in (0, 1)))
    keep = (first << 16 | second) >= below
    return torch.where(keep.reshape(x.shape), x * (2.0 ** 32 / (2 ** 32 - below)), 0.0)


def _norm(x, kind, weight, bias, eps=1e-6):
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + eps) * weight.float()
    return y if bias is None else y + bias.float()


def _plain(state):
    case = state["case"]
    x = state["x"].float()
    if case["op"] == "dropout":
        return dict(y=_drop(x, case["p"], state["random"], case["site"]).to(_type(case["stream"])))
    out = {}
    if case["op"] == "join":
        f = state["f"].float()
        if case["p"]:
            f = _drop(f, case["p"], state["random"], case["site"])
        if case["after"] != "none":
            f = _norm(f, case["after"], state["after_weight"], state.get("after_bias"))
        if case["gate"] != "none":
            f = f * state["gate"].float()
        x = case["skip_scale"] * x + case["branch_scale"] * f
        out["h"] = x.to(_type(case["stream"]))
    if case["before"] != "none":
        out["y"] = _norm(x, case["before"], state["before_weight"], state.get("before_bias")).to(_type(case["branch"]))
    return out


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own(state):
    from spiky_b200 import residual

    case = state["case"]
    if case["op"] == "dropout":
        return dict(y=residual.counter_dropout(state["x"], case["p"], state["random"], site=case["site"]))
    if case["op"] == "norm":
        return dict(y=residual.row_norm(state["x"], state["before_weight"], state.get("before_bias"), kind=case["before"], eps=1e-6,
                                        dtype=_type(case["branch"])))
    kind = {"none": None, "rms": "rms", "layer": "layer"}
    got = residual.residual_join(
        state["x"], state["f"], branch_norm=kind[case["after"]], branch_weight=state.get("after_weight"),
        branch_bias=state.get("after_bias"), gate=state.get("gate"), skip_scale=case["skip_scale"], branch_scale=case["branch_scale"],
        dropout=case["p"], state=state.get("random"), site=case["site"], next_norm=kind[case["before"]],
        next_weight=state.get("before_weight"), next_bias=state.get("before_bias"), eps=1e-6)
    return dict(h=got) if case["before"] == "none" else dict(h=got[0], y=got[1])


def run(state):
    if not state["case"]["train"]:
        with torch.no_grad():
            return _own(state) if own else _plain(state)
    out = _own(state) if own else _plain(state)
    names = state["leaves"]
    grads = torch.autograd.grad([out[k] for k in state["ups"]], [state[k] for k in names], [state["d" + k] for k in state["ups"]])
    result = {k: v.detach() for k, v in out.items()}
    result.update({"d" + k: g for k, g in zip(names, grads)})
    return result


def work(case):
    """Inputs read once and outputs written once; operations: about ten for each norm, four for gate and sum, twice that again backward."""
    n, width = case["sequences"] * case["length"] * case["width"], case["width"]
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    stream, branch, params = size[case["stream"]] * n, size[case["branch"]] * n, size[case["params"]]
    small = sum((1 + case["bias"]) * width * params for part in ("after", "before") if case[part] != "none")
    gate = {"none": 0, "width": width * params, "sequence": case["sequences"] * width * params, "element": branch}[case["gate"]]
    norms = (case["after"] != "none") + (case["before"] != "none")
    if case["op"] == "dropout":
        forward, backward = 2 * stream, 2 * stream
    elif case["op"] == "norm":
        forward, backward = stream + branch + small, branch + stream + small
    else:
        y = branch if case["before"] != "none" else 0
        forward, backward = 2 * stream + branch + y + gate + small, stream + y + stream + branch + gate + small
    flops = n * (2 + 10 * norms + 4 * (case["op"] == "join"))
    return dict(bytes=forward + (backward if case["train"] else 0), flops=flops * (3 if case["train"] else 1))


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_keep(p, random, site, n):
    """Which of n elements stay, products formed from 16-bit halves."""
    seed, offset = (int(v) % 2 ** 64 for v in random.tolist())
    offset = (offset + site) % 2 ** 64

    def product(c, m):   # (high, low) words of c * m; c a tensor or a number below 2^32
        low, high = (c & 0xFFFF) * m, (c >> 16) * m
        total = low + ((high & 0xFFFF) << 16)
        return (high >> 16) + (total >> 32), total & LOW32

    def digits(second):
        block = torch.arange((n + 7) // 8, dtype=torch.int64, device=DEVICE)
        word = [block % 2 ** 32, block // 2 ** 32 + second * 2 ** 31, offset % 2 ** 32, offset // 2 ** 32]
        key = [seed % 2 ** 32, seed // 2 ** 32]
        for r in range(10):
            h0, l0 = product(word[0], 0xD2511F53)
            h1, l1 = product(word[2], 0xCD9E8D57)
            word = [h1 ^ word[1] ^ ((key[0] + r * 0x9E3779B9) % 2 ** 32), l1, h0 ^ word[3] ^ ((key[1] + r * 0xBB67AE85) % 2 ** 32), l0]
        parts = torch.empty((block.numel(), 8), dtype=torch.int64, device=DEVICE)
        for k in range(4):
            parts[:, 2 * k], parts[:, 2 * k + 1] = word[k] % 2 ** 16, word[k] // 2 ** 16
        return parts.view(-1)[:n]

    return (digits(0) * 2 ** 16 + digits(1)) >= int(math.floor(p * 2.0 ** 32 + 0.5))


def _exact_norm(x, kind):
    """The normalised rows and the reciprocal deviation."""
    mean = x.mean(dim=-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    r = 1.0 / torch.sqrt((x - mean).pow(2).mean(dim=-1, keepdim=True) + 1e-6)
    return (x - mean) * r, r


def _exact_norm_back(u, xh, r, kind):
    """Gradient of a norm's input for the gradient u of its normalised rows."""
    v = u - xh * (u * xh).mean(dim=-1, keepdim=True)
    return r * (v - u.mean(dim=-1, keepdim=True) if kind == "layer" else v)


def exact(case, seed):
    state = prepare(case, seed)
    d = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v) and v.is_floating_point()}
    train, out = case["train"], {}
    drop = None
    if case["p"]:
        below = int(math.floor(case["p"] * 2.0 ** 32 + 0.5))
        drop = _exact_keep(case["p"], state["random"], case["site"], d["x"].numel()).view(d["x"].shape) * (2.0 ** 32 / (2 ** 32 - below))
    if case["op"] == "dropout":
        out["y"] = d["x"] * drop
        if train:
            out["dx"] = d["dy"] * drop
        return out
    h = d["x"]
    if case["op"] == "join":
        t = d["f"] if drop is None else d["f"] * drop
        n = t
        if case["after"] != "none":
            th, tr = _exact_norm(t, case["after"])
            n = th * d["after_weight"] + d.get("after_bias", 0.0)
        gate = d.get("gate", torch.ones((), dtype=torch.float64, device=DEVICE))
        h = case["skip_scale"] * d["x"] + case["branch_scale"] * gate * n
        out["h"] = h
    if case["before"] != "none":
        hh, hr = _exact_norm(h, case["before"])
        out["y"] = hh * d["before_weight"] + d.get("before_bias", 0.0)
    if not train:
        return out
    dh = d.get("dh", 0.0)
    if case["before"] != "none":
        out["dbefore_weight"] = (d["dy"] * hh).sum(dim=(0, 1))
        if case["bias"]:
            out["dbefore_bias"] = d["dy"].sum(dim=(0, 1))
        dh = dh + _exact_norm_back(d["dy"] * d["before_weight"], hh, hr, case["before"])
    out["dx"] = dh
    if case["op"] == "join":
        out["dx"] = case["skip_scale"] * dh
        dh = case["branch_scale"] * dh
        if case["gate"] != "none":
            sums = {"width": (0, 1), "sequence": (1,), "element": ()}[case["gate"]]
            out["dgate"] = (dh * n).sum(dim=sums, keepdim=case["gate"] == "sequence") if sums else dh * n
            dh = dh * gate
        if case["after"] != "none":
            out["dafter_weight"] = (dh * th).sum(dim=(0, 1))
            if case["bias"]:
                out["dafter_bias"] = dh.sum(dim=(0, 1))
            dh = _exact_norm_back(dh * d["after_weight"], th, tr, case["after"])
        out["df"] = dh if drop is None else dh * drop
    return out
