"""CPU tests of how the token-head operators meet autograd: forward-mode tangents, tracing and transforms that would miss what the kernels
write, and what is kept for the backward.  The stand-in provider writes memory as the kernels do, without torch knowing."""
import os
import sys

import pytest
import torch
from torch.autograd import forward_ad

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (ROOT, os.path.join(ROOT, "tests")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

import token_cpu_provider as P  # noqa: E402


def _raw(t):
    if t is None:
        return None
    out = torch.empty(tuple(int(v) for v in t.shape), dtype=t.dtype)
    out.numpy()[...] = t.detach().numpy()
    return out


def _seen(t):
    return t.detach() if isinstance(t, torch.Tensor) else t


class _Raw:
    """The provider's results in memory that torch did not see being written."""

    linear_fwd = staticmethod(lambda *a: tuple(_raw(t) for t in P.linear_fwd(*map(_seen, a))))
    norm_gate_fwd = staticmethod(lambda *a: tuple(_raw(t) for t in P.norm_gate_fwd(*map(_seen, a))))

    @staticmethod
    def grad_clip(src, dst=None, max_norm=0.0, eps=1e-6):
        norm = P.grad_clip([t.detach() for t in src])
        for s, d in zip(src, dst or []):
            d.detach().numpy()[...] = (s.detach() * torch.clamp(max_norm / (norm + eps), max=1.0)).numpy()
        return norm


def _calls():
    from protein_clip_amd import ops
    g = torch.Generator().manual_seed(0)
    w, r = torch.randn(8, 8, generator=g), torch.randn(3, 8, generator=g)
    one = torch.ones(8)
    return {"linear_act": lambda x: ops.linear_act(x, w, activation="gelu", kernels=_Raw),
            "linear_act weight": lambda x: ops.linear_act(r, x.t() @ x, kernels=_Raw),
            "linear_act residual": lambda x: ops.linear_act(r, w, residual=x, kernels=_Raw),
            "norm_gate_residual": lambda x: ops.norm_gate_residual(x, after=(one, None), kernels=_Raw),
            "norm_gate_residual two outputs": lambda x: ops.norm_gate_residual(r, x, before=(None, None), kernels=_Raw)[1]}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", sorted(_calls()))
def test_tangents_are_refused_not_dropped(name, grad):
    call = _calls()[name]
    x = torch.randn(3, 8, generator=torch.Generator().manual_seed(1))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(call(x), call(x.clone()))   # no operand has a tangent: the level alone refuses nothing
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(x[None])


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", sorted(_calls()))
def test_traces_hold_the_operator(name):
    """A trace of a call gives the call's results on new inputs, with and without gradients wanted."""
    call = _calls()[name]
    for requires in (False, True):
        g = torch.Generator().manual_seed(2)
        traced = torch.jit.trace(call, (torch.randn(3, 8, generator=g).requires_grad_(requires),))
        x = torch.randn(3, 8, generator=g)
        torch.testing.assert_close(traced(x), call(x))


@pytest.mark.filterwarnings("ignore")
def test_clipping_is_refused_where_it_would_not_be_seen():
    from protein_clip_amd import ops
    v = torch.ones(4)
    for call in (lambda t: ops.grad_norm([t], kernels=_Raw), lambda t: ops.clip_grads([t], 1.0, kernels=_Raw), lambda t: ops.clip_grads([v.clone()], 1.0, out=[t], kernels=_Raw)):
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward_ad.make_dual(v.clone(), torch.ones(4)))
            call(v.clone())
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(lambda t: call(t.clone()), (v,))
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.vmap(call)(v[None])
    assert torch.equal(v, torch.ones(4)) and ops.grad_norm(iter([v]), kernels=_Raw).item() == 2


def _kept(y):
    """The tensors that a result's graph holds on to, those of its own function only."""
    return [t for t in y.grad_fn.saved_tensors if t is not None]


@pytest.mark.parametrize("activation,res", [("none", False), ("relu", False), ("relu", True), ("gelu", True)])
def test_linear_keeps_what_its_gradients_read(activation, res):
    """x for the weight's gradient, the weight for the input's, the slope or the output for any; a frozen operand's partner may change."""
    from protein_clip_amd import ops
    for mask in range(1, 8):
        x, w, b = (torch.ones(*s).requires_grad_(bool(mask >> i & 1)) for i, s in enumerate(((3, 8), (4, 8), (4,))))
        y = ops.linear_act(x, w, b, torch.ones(3, 4) if res else None, activation=activation, kernels=P)
        kept = _kept(y)
        assert any(t is x for t in kept) == bool(mask & 2) and any(t is w for t in kept) == bool(mask & 1)
        assert len(kept) == bool(mask & 1) + bool(mask & 2) + (activation != "none")
        with torch.no_grad():
            if not mask & 2:
                x.add_(1)
            if not mask & 1:
                w.add_(1)
        grads = torch.autograd.grad(y.sum(), [v for v in (x, w, b) if v.requires_grad])
        assert [g.shape for g in grads] == [v.shape for v in (x, w, b) if v.requires_grad]


def test_bias_gradients_alone_on_the_host():
    """Which operands the kernels' wrapper wants for which gradient, refused before anything is launched."""
    from protein_clip_amd import kernels
    from protein_clip_amd._lib import PclipError
    x, w, dy = torch.ones(3, 8), torch.ones(4, 8), torch.ones(3, 4)
    for args, want in (((None, w, dy), (True, True, True)), ((x, None, dy), (True, False, False)), ((None, None, dy), (False, False, True)), ((None, w, dy), (True, False, True)),
                       ((None, torch.ones(5, 8), dy), (True, False, False))):
        with pytest.raises(PclipError):
            kernels.linear_bwd(*args, want_dx=want[0], want_dw=want[1], want_db=want[2])


@pytest.mark.parametrize("after", [None, "norm"])
@pytest.mark.parametrize("before", [None, "norm"])
@pytest.mark.parametrize("gate", [None, "mask", "learned"])
def test_norm_gate_keeps_what_its_gradients_read(after, before, gate):
    """The residual only for the second norm; the block's output only where a norm or the gate's gradient reads it.  What is not kept may be
    changed in place before the backward."""
    from protein_clip_amd import ops
    g = torch.Generator().manual_seed(3)
    make = lambda: torch.randn(5, 8, generator=g)
    u, r, dy, dn = make().requires_grad_(True), make().requires_grad_(True), make(), make()
    gt = {None: None, "mask": make() > 0, "learned": torch.randn(8, generator=g).requires_grad_(True)}[gate]
    w = torch.randn(8, generator=g).requires_grad_(True)
    pair = lambda on: None if on is None else (w, None)
    want = P._norm_gate(u, r, gt, 1 if gate != "learned" else 5, 0.5, after and "layer", w, None, before and "layer", w, None, 1e-5)
    leaves = [t for t in (u, r, gt, w) if t is not None and t.requires_grad and (t is not w or after or before)]
    cot = (dy, dn) if before else (dy,)
    refs = torch.autograd.grad([o for o in want if o is not None], leaves, cot)
    outs = ops.norm_gate_residual(u, r, gt, scale=0.5, after=pair(after), before=pair(before), kernels=P)
    outs = outs if before else (outs,)
    kept = _kept(outs[0])
    assert any(t is r for t in kept) == bool(before)
    assert any(t is u for t in kept) == bool(after or before or gate == "learned")
    with torch.no_grad():
        if not before:
            r.add_(1)
        if not (after or before or gate == "learned"):
            u.add_(1)
    for got, ref in zip(torch.autograd.grad(outs, leaves, cot), refs):
        torch.testing.assert_close(got, ref, rtol=1e-4, atol=1e-5)


class _Strict(_Raw):
    """Takes what the kernels take: a destination of its source's layout, without gaps."""

    @staticmethod
    def grad_clip(src, dst=None, max_norm=0.0, eps=1e-6):
        from protein_clip_amd import kernels
        for s, d in zip(src, dst or []):
            assert kernels._dense(s) and kernels._dense(d) and s.shape == d.shape and (s.stride() == d.stride() or s.is_contiguous() and d.is_contiguous())
        return _Raw.grad_clip(src, dst, max_norm, eps)


def test_summed_gradients_of_any_layout_are_clipped(monkeypatch):
    """The way back from the flat buffer of the sum over ranks: with a limit, gradients of every layout that it fills without one, also those
    with gaps, and the norm is the sum's."""
    from protein_clip_amd import ops
    from protein_clip_amd.modules import training_utils as U
    monkeypatch.setattr(ops, "_hip_kernels", _Strict)
    monkeypatch.setattr(U.dist, "all_reduce", lambda t, group=None: t.mul_(2))   # two ranks with the same gradients

    def model():
        g = torch.Generator().manual_seed(0)
        m = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(s)) for s in ((6, 4), (3, 2, 5), (7,), (4, 4), (5,))])
        for p, lay in zip(m, (lambda v: v.t().contiguous().t(), lambda v: v.permute(2, 0, 1).contiguous().permute(1, 2, 0), lambda v: v, lambda v: torch.stack([v, v], 2)[:, :, 0],
                              lambda v: v)):
            p.grad = lay(torch.randn(p.shape, generator=g))
        return m

    free, clipped = model(), model()
    strides = [p.grad.stride() for p in clipped]
    U._sum_head_grads(free)
    U._sum_head_grads(clipped, max_grad_norm=0.5)
    size = torch.sqrt(sum((p.grad.double() ** 2).sum() for p in free)).item()
    for p, q, st in zip(free, clipped, strides):
        torch.testing.assert_close(q.grad, p.grad * (0.5 / size), rtol=1e-5, atol=1e-7)
        assert q.grad.stride() == st


def test_clip_grad_norm_takes_no_third_argument_by_position():
    """torch's own function has the norm's type there: a call written for it must not set eps in silence."""
    from protein_clip_amd import ops
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    with pytest.raises(TypeError):
        ops.clip_grad_norm_([p], 1.0, 2.0, kernels=_Raw)
    assert torch.equal(p.grad, torch.ones(4))
    assert ops.clip_grad_norm_([p], 1.0, eps=0.0, error_if_nonfinite=True, kernels=_Raw).item() == 2 and torch.equal(p.grad, torch.full((4,), 0.5))
