"""Plain 64-bit forms of the token-head operators and the bounds their GPU results are held to.

Bounds.  ``half(t)`` is half a step of a type relative to the value, ``floor(t)`` half the smallest subnormal (what a
rounding to zero may lose).  A 32-bit addition or product is off by at most 2^-24 of its result; the matrix cores'
additions are counted with a whole step, 2^-23."""
import torch

F64 = torch.float64
U = 2.0 ** -23


def half(t):
    return torch.finfo(t).eps / 2


def floor(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


def rounded(ref, err, t):
    """Bound of a value known to ``err`` after one rounding to ``t``."""
    return err + half(t) * (ref.abs() + err) + floor(t)


def assert_within(got, ref, tol, what):
    got, ref = got.detach().cpu().to(F64), ref.to(F64)
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} instead of {tuple(ref.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - ref).abs() - tol
    assert (over <= 0).all(), f"{what}: off by {(got - ref).abs().flatten()[over.argmax()]:.3e}, allowed {tol.expand_as(ref).flatten()[over.argmax()]:.3e}"


# ---- linear ---------------------------------------------------------------------------------------------
def act(z, name):
    """(value, slope) of the activation."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def linear(x, w, b, r, name):
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = act(z, name)[0]
    return y if r is None else y + r


def linear_bounds(x, w, b, r, dy, name, t, grads=True):
    """{"y", "x", "weight", "bias"}: (value, bound) of the forward and of the gradients, operands in 64 bits holding values of type
    ``t``.  z is a sum of K products and the bias: K + 1 additions.  Activations are 1.13-Lipschitz with slopes that are 1-Lipschitz,
    and computed to 4e-6 of the value in 16-bit types (fitted Gaussian tail, hardware exp and reciprocal), to 1e-6 in f32.  dz carries
    the rounding of the slope (gelu, silu) and its own."""
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    size = x.abs() @ w.abs().t() + (0 if b is None else b.abs())
    z = linear(x, w, b, None, "none")
    ez = (K + 1) * U * size
    y, slope = act(z, name)
    approx = 0.0 if name in ("none", "relu") else (1e-6 if t == torch.float32 else 4e-6)
    ey = 1.13 * ez + approx * (y.abs() + z.abs())
    full = y if r is None else y + r
    out = {"y": (full, rounded(full, ey + U * full.abs(), t))}
    if not grads:
        return out
    smooth = name in ("gelu", "silu")
    es = (ez + approx + half(t) + floor(t)) if smooth else (z.abs() <= ez).to(F64) if name == "relu" else torch.zeros_like(z)
    dz = dy * slope
    edz = dy.abs() * es
    if name != "none":
        edz = edz + half(t) * (dz.abs() + edz) + floor(t)
    sums = lambda value, err, size, n: (value, rounded(value, err + (n + 8) * U * (size + err), t))
    out["x"] = sums(dz @ w, edz @ w.abs(), dz.abs() @ w.abs(), N)
    out["weight"] = sums(dz.t() @ x, edz.t() @ x.abs(), dz.abs().t() @ x.abs(), M)
    out["bias"] = sums(dz.sum(0), edz.sum(0), dz.abs().sum(0), M)
    return out


# ---- norms around a block ----------------------------------------------------------------------------------
def normed(v, kind, w, b, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v if w is None else v * w
    return v if b is None else v + b


def norm_gate(u, r, gate, scale, after, before, kind, eps=1e-5):
    """``gate`` broadcastable to u; ``after`` / ``before`` None or (weight, bias)."""
    y = u if after is None else normed(u, kind, after[0], after[1], eps)
    if gate is not None:
        y = y * gate
    y = y * scale
    if r is not None:
        y = y + r
    return (y,) if before is None else (y, normed(y, kind, before[0], before[1], eps))


def _stats(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = torch.rsqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    # what a rounding of v or of its mean is worth in units of the normalised value
    return (v - mean) * rstd, rstd, 1 + rstd * (v.abs() + v.abs().mean(-1, keepdim=True)).amax(-1, keepdim=True)


ROUNDINGS = 64 * U   # a row's sum: 16 additions in a lane, 8 halving steps; two such sums and a few products a norm


def norm_gate_bounds(u, r, gate, scale, after, before, kind, dy, dn, t, eps=1e-5):
    """{"y", "n", "u", "residual", "gate" (per element), "wa", "ba", "wb", "bb"}: (value, bound).  The bound of each value is the
    roundings of its formula (ROUNDINGS for each norm or its derivative) times the formula evaluated with every term's absolute
    value, times what an error of a normalised value's input is worth."""
    one = torch.ones_like(u)
    g = one if gate is None else gate.expand_as(u)
    wa = one if after is None or after[0] is None else after[0]
    ba = 0 * one if after is None or after[1] is None else after[1]
    wb = one if before is None or before[0] is None else before[0]
    ka, kb = one[..., :1], one[..., :1]
    v, ev = u, 0 * u
    if after is not None:
        ha, sa, ka = _stats(u, kind, eps)
        v = ha * wa + ba
        ev = ROUNDINGS * ka * (1 + ha.abs()) * wa.abs() + U * (v.abs() + ba.abs())
    y = scale * g * v + (0 if r is None else r)
    ey = scale * g.abs() * ev + 4 * U * ((scale * g * v).abs() + y.abs())
    out = {"y": (y, rounded(y, ey, t))}
    edt = 0 * u
    dt = 0 * u if dy is None else dy
    if before is not None:
        hb, sb, kb = _stats(y, kind, eps)
        n = hb * wb + (0 if before[1] is None else before[1])
        # the error of y moves the normalised value by at most rstd * (its own + the row's largest twice)
        eh = ROUNDINGS * kb * (1 + hb.abs()) + sb * (ey + (1 + hb.abs()) * ey.amax(-1, keepdim=True))
        out["n"] = (n, rounded(n, eh * wb.abs() + 2 * U * n.abs() + (0 if before[1] is None else U * before[1].abs()), t))
        if dn is not None:
            d = dn * wb
            m = d.abs().mean(-1, keepdim=True)
            back = sb * (d - hb * (d * hb).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0))
            worst = eh.amax(-1, keepdim=True)
            size = sb * (d.abs() + m + hb.abs() * (d * hb).abs().mean(-1, keepdim=True))
            edt = ROUNDINGS * kb * size + sb * (eh * (d * hb).abs().mean(-1, keepdim=True) + hb.abs() * worst * m) + 4 * worst * size
            dt = dt + back
            out["wb"] = (dn * hb, dn.abs() * eh + U * (dn * hb).abs())
            out["bb"] = (dn, 0 * dn)
    edt = edt + U * dt.abs()
    out["residual"] = (dt, rounded(dt, edt, t))
    out["gate"] = (scale * v * dt, scale * (v.abs() * edt + ev * dt.abs()) + 4 * U * (scale * v * dt).abs())
    dv, edv = scale * g * dt, scale * g.abs() * edt + 2 * U * (scale * g * dt).abs()
    du, edu = dv, edv
    if after is not None:
        eh = ROUNDINGS * ka * (1 + ha.abs())
        worst = eh.amax(-1, keepdim=True)
        out["wa"] = (dv * ha, edv * ha.abs() + dv.abs() * eh + U * (dv * ha).abs())
        out["ba"] = (dv, edv)
        d, ed = dv * wa, edv * wa.abs()
        mean = lambda q: q.mean(-1, keepdim=True)
        du = sa * (d - ha * mean(d * ha) - (mean(d) if kind == "layer" else 0))
        size = sa * (d.abs() + mean(d.abs()) + ha.abs() * mean((d * ha).abs()))
        edu = ROUNDINGS * ka * size + sa * (ed + mean(ed) + ha.abs() * mean(ed * ha.abs()) + eh * mean((d * ha).abs()) + ha.abs() * worst * mean(d.abs())) + 4 * worst * size
    out["u"] = (du, rounded(du, edu, t))
    return out


def column_sum(value, err, t, rows, dims):
    """A sum over ``rows`` rows, at most one addition each in 32 bits, rounded to ``t``."""
    s = value.sum(dims)
    return s, rounded(s, err.sum(dims) + (rows + 32) * U * (value.abs() + err).sum(dims), t)
