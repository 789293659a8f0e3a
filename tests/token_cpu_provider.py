"""``cpu_provider`` (the test-only stand-in for the kernel provider) with the token-head operators added, in plain torch."""
import torch

import token_ref as R
from cpu_provider import *  # noqa: F401,F403


def linear_fwd(x, w, bias=None, residual=None, activation="none", want_slope=False):
    z = R.linear(x, w, bias, None, "none")
    y, slope = R.act(z, activation)
    return (y if residual is None else y + residual), (slope if want_slope else None)


def linear_bwd(x, w, dy, saved=None, saved_is_output=False, activation="none", want_dx=True, want_dw=True, want_db=True):
    flat = lambda t: t.reshape(-1, t.shape[-1])
    dz = dy if saved is None else dy * ((saved > 0).to(dy.dtype) if saved_is_output else saved)
    return (dz @ w if want_dx else None), (flat(dz).t() @ flat(x) if want_dw else None), (flat(dz).sum(0) if want_db else None)


def _norm_gate(u, r, gate, gate_rows, scale, after, wa, ba, before, wb, bb, eps):
    g = None if gate is None else gate.to(u.dtype).reshape(-1, u.shape[-1]).repeat_interleave(gate_rows, 0).reshape(u.shape)
    return R.norm_gate(u, r, g, scale, (wa, ba) if after else None, (wb, bb) if before else None, after or before, eps)


def norm_gate_fwd(u, r=None, gate=None, gate_rows=1, scale=1.0, after=None, wa=None, ba=None, before=None, wb=None, bb=None, eps=1e-5,
                  want_stats=False):
    out = _norm_gate(u, r, gate, gate_rows, scale, after, wa, ba, before, wb, bb, eps)
    return out[0], (out[1] if before else None), None


def norm_gate_bwd(u, r, gate, gate_rows, scale, after, wa, ba, before, wb, bb, eps, stats, dy, dn, want=(True,) * 7):
    operands = (u, r, gate, wa, ba, wb, bb)
    leaves = [t.detach().clone().requires_grad_(w) if t is not None else None for t, w in zip(operands, want)]
    with torch.enable_grad():
        outs = _norm_gate(*leaves[:3], gate_rows, scale, after, leaves[3], leaves[4], before, leaves[5], leaves[6], eps)
        total = sum((o * d).sum() for o, d in zip(outs, (dy, dn)) if d is not None)
        grads = iter(torch.autograd.grad(total, [t for t in leaves if t is not None and t.requires_grad], allow_unused=True))
    return tuple(next(grads) if t is not None and t.requires_grad else None for t in leaves)


def grad_clip(src, dst=None, max_norm=0.0, eps=1e-6):
    norm = torch.sqrt(sum((t.double() ** 2).sum() for t in src)).float().reshape(1)
    if dst is not None:
        factor = torch.clamp(max_norm / (norm[0] + eps), max=1.0)
        for s, d in zip(src, dst):
            d.copy_(s * factor)
    return norm
