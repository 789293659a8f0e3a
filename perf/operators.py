"""What is measured of the token-head operators: the linear layer with bias, activation and residual in its
epilogue, the norms around a block with its gate, scale and residual, and the global gradient norm with clipping.

``listed()`` names the cases, ``draw`` makes more of the same ranges, ``prepare`` makes the inputs of one, ``run``
is one pass (the plain torch form, or the framework's operators where ``own`` is true), ``exact`` the same in 64
bits, and ``work`` what a pass cannot do without.

The sizes are the towers' own: 640 is the trunk's width, 2560 its feed-forward width, 128 the embedding width,
65,536 tokens a batch of 256 sequences of 256 tokens."""
import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def _linear(rows, width, out, dtype, pass_, activation="none", bias=True, residual=False, frozen=False):
    """``pass_``: "forward" (inference) or "train" (forward and every gradient); ``frozen``: the input comes from a
    frozen trunk and takes no gradient."""
    return {"op": "linear", "rows": rows, "width": width, "out": out, "dtype": dtype, "pass": pass_, "activation": activation, "bias": bias,
            "residual": residual, "frozen": frozen}


def _norm(batch, tokens, width, dtype, pass_, gate="none", after="none", before="none", kind="layer", residual=True, scale=1.0):
    """``after`` / ``before``: "none", "plain" (no affine) or "affine"; ``gate``: "none", "channel" [width],
    "sequence" [batch,1,width], "element" [batch,tokens,width] or "keep" (a dropout mask of bytes)."""
    return {"op": "norm", "batch": batch, "tokens": tokens, "width": width, "dtype": dtype, "pass": pass_, "gate": gate, "after": after,
            "before": before, "kind": kind, "residual": residual, "scale": scale}


def _clip(layout, source, target, max_norm, tensors=0, elements=0, pick=0):
    """``layout``: "heads" (the trainable tensors of both towers), "trunk" (every tensor of the 30-layer trunk) or
    "ragged" (``tensors`` tensors of ``elements`` elements in all, sizes picked by ``pick``)."""
    return {"op": "clip", "layout": layout, "source": source, "target": target, "max_norm": max_norm, "tensors": tensors, "elements": elements,
            "pick": pick}


def listed():
    named = [
        # scoring one peptide: 29 residues with their two special tokens, through the projection
        ("linear-one-peptide", _linear(31, 640, 128, "bf16", "forward")),
        # the projection behind the frozen trunk in a training step of 16 pairs, in the type of the reference's run
        ("linear-projection-f32", _linear(4096, 640, 128, "f32", "train", frozen=True)),
        # the per-residue feed-forward layer over a batch of 256 sequences of 256 tokens
        ("linear-residue-relu", _linear(65536, 128, 128, "bf16", "train", "relu")),
        # the first layer of a trunk block's feed-forward part, trained on a full batch: the largest case
        ("linear-trunk-up", _linear(65536, 640, 2560, "bf16", "train", "gelu")),
        # its second layer with the residual stream, while embeddings are computed for a search
        ("linear-trunk-down", _linear(16384, 2560, 640, "bf16", "forward", residual=True)),
        # sizes that divide by nothing: the last batch of an epoch through a head of odd widths
        ("linear-ragged", _linear(4999, 637, 331, "f16", "train", "silu", residual=True)),
        # LayerNorm and dropout of the per-residue feed-forward layer, in training
        ("norm-residue-dropout", _norm(256, 256, 128, "bf16", "train", gate="keep", after="affine", residual=False, scale=1.0 / 0.9)),
        # the join of two trunk blocks with a gate for each sequence (a conditioned block), in training
        ("norm-block-join", _norm(64, 512, 640, "bf16", "train", gate="sequence", after="affine", before="affine", kind="rms", scale=0.5)),
        # the same join for one token of inference, without a gate
        ("norm-one-token", _norm(1, 1, 640, "bf16", "forward", before="affine")),
        # odd width and length in 32 bits with a learned scale for each channel
        ("norm-ragged", _norm(3, 1001, 1283, "f32", "train", gate="channel", after="affine", before="affine", scale=0.25)),
        # clipping the towers' own gradients: some thirty small tensors, where latency counts
        ("clip-heads", _clip("heads", "f32", "f32", 1.0)),
        # clipping when the whole trunk is trained: bfloat16 sums into the 32-bit gradients of the optimizer
        ("clip-trunk", _clip("trunk", "bf16", "f32", 1.0)),
    ]
    return [dict(case, name=name) for name, case in named]


def _spread(rng, low, high):
    """A whole number between the two, spread evenly over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "clip"])
    pass_ = rng.choice(["forward", "train", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "linear":
        size = lambda: rng.choice([128, 320, 640, 1280, 2560, _spread(rng, 8, 2560), _spread(rng, 8, 2560)])
        width, out = size(), size()
        rows = _spread(rng, 1, min(65536 if dtype != "f32" else 16384, 65536 * 640 * 2560 // (width * out)))   # no dearer than the largest listed
        return _linear(rows, width, out, dtype, pass_, rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.8, rng.random() < 0.4,
                       pass_ == "train" and rng.random() < 0.25)
    if op == "norm":
        gate = rng.choice(["none", "channel", "sequence", "element", "keep"])
        after = rng.choice(["affine", "affine", "plain", "none"])
        before = rng.choice(["affine", "plain", "none"])
        return _norm(_spread(rng, 1, 64), _spread(rng, 1, 512), rng.choice([128, 320, 640, 1280, _spread(rng, 8, 2560), _spread(rng, 8, 2560)]), dtype, pass_,
                     gate, after, before, rng.choice(["layer", "rms"]), rng.random() < 0.7, rng.choice([1.0, 0.5, 1.0 / 0.9]))
    source, target = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
    tensors = _spread(rng, 1, 600)
    return _clip("ragged", source, target, rng.choice([1.0, 0.1, 1e6]), tensors, max(tensors, _spread(rng, 1000, 60_000_000)), rng.randrange(1 << 20))


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def _clip_sizes(case):
    if case["layout"] == "heads":
        block = [(128, 128), (128,), (128,), (128,), (128, 128), (128,)]          # Linear, LayerNorm, Linear
        return ([(128, 640), (128,)] + block + block) * 2 + [(1,)]
    if case["layout"] == "trunk":
        layer = [(640, 640), (640,)] * 4 + [(640,)] * 4 + [(2560, 640), (2560,), (640, 2560), (640,)]
        return [(33, 640), (1026, 640)] + layer * 30 + [(640,), (640,)]
    pick = random.Random(case["pick"])
    shares = [math.exp(pick.uniform(0.0, 9.0)) for _ in range(case["tensors"])]
    total = sum(shares)
    return [(max(1, int(case["elements"] * s / total)),) for s in shares]


def _inputs(case, seed):
    """The tensors of a case, in their own types, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]] if "dtype" in case else None

    def normal(*shape, std=1.0, mean=0.0, dt=None):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt or dtype)

    if case["op"] == "linear":
        rows, width, out = case["rows"], case["width"], case["out"]
        bound = 1.0 / math.sqrt(width)   # the initial spread of a linear layer's weights
        t = {"x": normal(rows, width), "weight": ((torch.rand(out, width, generator=g, device="cuda") * 2 - 1) * bound).to(dtype)}
        if case["bias"]:
            t["bias"] = ((torch.rand(out, generator=g, device="cuda") * 2 - 1) * bound).to(dtype)
        if case["residual"]:
            t["residual"] = normal(rows, out)
        if case["pass"] == "train":
            t["dy"] = normal(rows, out)
        return t
    if case["op"] == "norm":
        batch, tokens, width = case["batch"], case["tokens"], case["width"]
        t = {"u": normal(batch, tokens, width, std=1.5, mean=0.25)}
        if case["residual"]:
            t["residual"] = normal(batch, tokens, width, std=2.0)
        if case["gate"] == "keep":
            t["gate"] = (torch.rand(batch, tokens, width, generator=g, device="cuda") >= 0.1).to(torch.uint8)
        elif case["gate"] != "none":
            shape = {"channel": (width,), "sequence": (batch, 1, width), "element": (batch, tokens, width)}[case["gate"]]
            t["gate"] = normal(*shape, std=0.5, mean=0.5)
        for which in ("after", "before"):
            if case[which] == "affine":
                t[which + "_weight"] = normal(width, std=0.1, mean=1.0, dt=torch.float32)
                if case["kind"] == "layer":
                    t[which + "_bias"] = normal(width, std=0.1, dt=torch.float32)
        if case["pass"] == "train":
            t["dy"] = normal(batch, tokens, width)
            if case["before"] != "none":
                t["dn"] = normal(batch, tokens, width)
        return t
    spread = 10.0 ** (torch.rand(1, generator=g, device="cuda").item() - 2.0)   # what a step's gradients measure varies
    return {"source": [normal(*s, std=spread, dt=_DTYPES[case["source"]]) for s in _clip_sizes(case)]}


_NO_GRADIENT = ("dy", "dn")


def _leaves(case, t):
    """Names of the inputs that take a gradient, in the order in which the gradients are returned."""
    skip = set(_NO_GRADIENT)
    if case.get("frozen"):
        skip.add("x")
    if case.get("gate") == "keep":
        skip.add("gate")
    return [n for n in t if n not in skip]


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if case["op"] == "clip":
        # the optimizer's gradients are views of one flat buffer, as a trainer that sums them over ranks keeps them
        sizes = [s.numel() for s in t["source"]]
        state["flat"] = torch.zeros(sum(sizes), dtype=_DTYPES[case["target"]], device="cuda")
        state["target"] = [v.view_as(s) for v, s in zip(state["flat"].split(sizes), t["source"])]
    elif case["pass"] == "train":
        state["leaves"] = _leaves(case, t)
        for n in state["leaves"]:
            t[n].requires_grad_(True)
    if own:
        import protein_clip_amd  # noqa: F401
        from protein_clip_amd import ops
        state["ops"] = ops
    return state


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def _activate(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * (1.0 / math.sqrt(2.0))))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_linear(t, case):
    z = t["x"].float() @ t["weight"].float().t()
    if "bias" in t:
        z = z + t["bias"].float()
    y = _activate(z, case["activation"])
    if "residual" in t:
        y = y + t["residual"].float()
    return (y.to(t["x"].dtype),)


def _plain_normed(v, kind, weight, bias, eps=1e-5):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    if weight is not None:
        v = v * weight
    if bias is not None:
        v = v + bias
    return v


def _plain_norm(t, case):
    dtype = t["u"].dtype
    y = t["u"].float()
    if case["after"] != "none":
        y = _plain_normed(y, case["kind"], t.get("after_weight"), t.get("after_bias"))
    if "gate" in t:
        y = y * t["gate"].float()
    y = y * case["scale"]
    if "residual" in t:
        y = y + t["residual"].float()
    if case["before"] == "none":
        return (y.to(dtype),)
    return y.to(dtype), _plain_normed(y, case["kind"], t.get("before_weight"), t.get("before_bias")).to(dtype)


def _plain_clip(source, target, max_norm, eps=1e-6):
    norm = torch.sqrt(torch.stack([(s.double() * s.double()).sum() for s in source]).sum()).float()
    factor = torch.clamp(max_norm / (norm + eps), max=1.0)
    for s, d in zip(source, target):
        d.copy_(s.float() * factor)
    return norm


def _own_linear(ops, t, case):
    return (ops.linear_act(t["x"], t["weight"], t.get("bias"), t.get("residual"), activation=case["activation"]),)


def _own_norm(ops, t, case):
    affine = lambda which: None if case[which] == "none" else (t.get(which + "_weight"), t.get(which + "_bias"))
    out = ops.norm_gate_residual(t["u"], t.get("residual"), t.get("gate"), scale=case["scale"], after=affine("after"), before=affine("before"),
                                 norm=case["kind"])
    return out if isinstance(out, tuple) else (out,)


def run(state):
    case, t = state["case"], state["t"]
    if case["op"] == "clip":
        if own:
            norm = state["ops"].clip_grads(t["source"], case["max_norm"], out=state["target"])
        else:
            norm = _plain_clip(t["source"], state["target"], case["max_norm"])
        return [norm, state["flat"]]
    if own:
        outs = (_own_linear if case["op"] == "linear" else _own_norm)(state["ops"], t, case)
    else:
        outs = (_plain_linear if case["op"] == "linear" else _plain_norm)(t, case)
    if case["pass"] == "forward":
        return list(outs)
    grads = torch.autograd.grad(outs, [t[n] for n in state["leaves"]], [t[n] for n in _NO_GRADIENT if n in t])
    return [o.detach() for o in outs] + list(grads)


# ---------------------------------------------------------------------------------------------------------
# the same in 64 bits, from the formulas
# ---------------------------------------------------------------------------------------------------------
def _exact_linear(case, t):
    x, w = t["x"].double(), t["weight"].double()
    z = torch.mm(x, w.t().contiguous())
    if "bias" in t:
        z += t["bias"].double()
    kind = case["activation"]
    if kind == "relu":
        y, slope = z.clamp(min=0), (z > 0).double()
    elif kind == "gelu":
        phi = torch.special.ndtr(z)
        y, slope = z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    elif kind == "silu":
        s = torch.sigmoid(z)
        y, slope = z * s, s + z * s * (1.0 - s)
    else:
        y, slope = z, None
    if "residual" in t:
        y = y + t["residual"].double()
    if case["pass"] == "forward":
        return [y]
    dy = t["dy"].double()
    dz = dy if slope is None else dy * slope
    of = {"x": lambda: torch.mm(dz, w), "weight": lambda: torch.mm(dz.t().contiguous(), x), "bias": lambda: dz.sum(0), "residual": lambda: dy}
    return [y] + [of[n]() for n in _leaves(case, t)]


def _exact_normed(v, kind, weight, bias):
    """(normalised and affine value, what the gradient needs)"""
    centre = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    spread = 1.0 / torch.sqrt(((v - centre) ** 2).mean(-1, keepdim=True) + 1e-5)
    hat = (v - centre) * spread
    out = hat if weight is None else hat * weight.double()
    return (out if bias is None else out + bias.double()), hat, spread


def _exact_normed_back(d, hat, spread, kind, weight):
    dims = tuple(range(d.dim() - 1))
    dweight, dbias = (d * hat).sum(dims), d.sum(dims)
    dh = d if weight is None else d * weight.double()
    dv = dh - hat * (dh * hat).mean(-1, keepdim=True)
    if kind == "layer":
        dv = dv - dh.mean(-1, keepdim=True)
    return dv * spread, dweight, dbias


def _exact_norm(case, t):
    kind, scale = case["kind"], case["scale"]
    u = t["u"].double()
    v = u
    if case["after"] != "none":
        v, hat_a, spread_a = _exact_normed(u, kind, t.get("after_weight"), t.get("after_bias"))
    gate = t["gate"].double() if "gate" in t else torch.ones((), dtype=torch.float64, device=u.device)
    y = v * gate * scale
    if "residual" in t:
        y = y + t["residual"].double()
    outs = [y]
    if case["before"] != "none":
        n, hat_b, spread_b = _exact_normed(y, kind, t.get("before_weight"), t.get("before_bias"))
        outs.append(n)
    if case["pass"] == "forward":
        return outs
    g = {}
    dy = t["dy"].double()
    if case["before"] != "none":
        more, g["before_weight"], g["before_bias"] = _exact_normed_back(t["dn"].double(), hat_b, spread_b, kind, t.get("before_weight"))
        dy = dy + more
    g["residual"] = dy
    dgate = dy * v * scale
    if "gate" in t:
        g["gate"] = {"channel": lambda: dgate.sum((0, 1)), "sequence": lambda: dgate.sum(1, keepdim=True)}.get(case["gate"], lambda: dgate)()
    dv = dy * gate * scale
    if case["after"] != "none":
        dv, g["after_weight"], g["after_bias"] = _exact_normed_back(dv, hat_a, spread_a, kind, t.get("after_weight"))
    g["u"] = dv
    return outs + [g[n] for n in _leaves(case, t)]


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, t)
    if case["op"] == "norm":
        return _exact_norm(case, t)
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(s.double())) ** 2 for s in t["source"]))
    factor = min(1.0, case["max_norm"] / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64, device="cuda"), torch.cat([s.double().reshape(-1) for s in t["source"]]) * factor]


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "linear":
        m, k, n, b = case["rows"], case["width"], case["out"], _BYTES[case["dtype"]]
        vec = n if case["bias"] else 0
        res = m * n if case["residual"] else 0
        nbytes, flops = (m * k + n * k + vec + res + m * n) * b, 2 * m * k * n
        if case["pass"] == "train":   # dy in; the gradients out; one product for each operand's gradient
            dx = 0 if case["frozen"] else m * k
            nbytes += (m * n + dx + n * k + vec + res) * b
            flops *= 2 if case["frozen"] else 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "norm":
        rows, d, b = case["batch"] * case["tokens"], case["width"], _BYTES[case["dtype"]]
        e = rows * d
        gate = {"none": 0, "channel": d * b, "sequence": case["batch"] * d * b, "element": e * b, "keep": e}[case["gate"]]
        res = e * b if case["residual"] else 0
        affine = sum(d * 4 * (2 if case["kind"] == "layer" else 1) for which in ("after", "before") if case[which] == "affine")
        outs = e * b * (2 if case["before"] != "none" else 1)
        nbytes = e * b + gate + res + affine + outs
        if case["pass"] == "train":
            nbytes += outs + e * b + res + affine + (0 if case["gate"] == "keep" else gate)
        return {"bytes": nbytes, "flops": e * (60 if case["pass"] == "train" else 20)}
    count = sum(math.prod(s) for s in _clip_sizes(case))
    return {"bytes": count * (_BYTES[case["source"]] + _BYTES[case["target"]]) + 4, "flops": 3 * count}
