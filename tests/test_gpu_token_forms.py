"""GPU tests of the kernels that large linear layers and the other widths of the norms run on, against 64-bit forms computed on the GPU."""
import pytest
import torch

import test_gpu_token_ops as T
import token_forms as F
import token_ref as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = T.F32, T.BF16, T.F16
ops = T.ops


def _make(g, t, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)


@pytest.mark.parametrize("t", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rows,width,out,name,has_bias,has_res,tiles,aligned", F.LINEAR)
def test_linear_forms(ops, t, rows, width, out, name, has_bias, has_res, tiles, aligned):
    """Every value within the bounds of token_ref, which grow with the lengths of the sums; and all together, in the 2-norm, within three half
    steps of the type: results are rounded once, dz once before, independently of each other.  4e-6 for the sums in f32; where ReLU's input
    is within their error of zero, a share of some 1e-6 of the units has the other slope, whose gradients change by the root of it."""
    g = torch.Generator(device="cuda").manual_seed(rows + out)
    x, w = _make(g, t, rows, width), _make(g, t, out, width, std=width ** -0.5)
    b = _make(g, t, out, std=0.3) if has_bias else None
    r = _make(g, t, rows, out) if has_res else None
    dy = _make(g, t, rows, out)
    wide = lambda v: None if v is None else v.double()
    want = R.linear_bounds(wide(x), wide(w), wide(b), wide(r), wide(dy), name, t)
    leaves = {"x": x, "weight": w} | ({"bias": b} if has_bias else {}) | ({"residual": r} if has_res else {})
    for v in leaves.values():
        v.requires_grad_(True)
    y = ops.linear_act(x, w, b, r, activation=name)
    got = {"y": y.detach()} | dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, r, activation=name), got["y"])
    if has_res:
        assert torch.equal(got.pop("residual"), dy)
    for n, v in got.items():
        ref, tol = want[n]
        R.assert_within(v, ref.cpu(), tol.cpu(), n)
        off = ((v.double() - ref).norm() / ref.norm()).item()
        assert off <= 3 * R.half(t) + 4e-6 + (1e-3 if name == "relu" and n != "y" else 0), f"{n}: {off:.2e} in the 2-norm"


@pytest.mark.parametrize("rows,width,out,name,has_bias,has_res,splits", F.SPLIT)
def test_split_products(ops, rows, width, out, name, has_bias, has_res, splits):
    """The split contraction like any other, the same bits on every call, and from the entry that takes no scratch the unsplit result."""
    from protein_clip_amd import _lib
    from protein_clip_amd._lib import ptr, stream_of
    test_linear_forms(ops, F32, rows, width, out, name, has_bias, has_res, None, None)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = _make(g, F32, rows, width), _make(g, F32, out, width, std=width ** -0.5)
    y = [ops.linear_act(x, w) for _ in range(2)]
    assert torch.equal(*y)
    unsplit = torch.empty_like(y[0])
    _lib.check(_lib.load().pclip_linear_fwd(ptr(x), ptr(w), None, None, rows, width, out, 0, 0, ptr(unsplit), None, stream_of(x)), "pclip_linear_fwd")
    size = x.double().abs() @ w.double().abs().t()
    assert ((unsplit.double() - y[0].double()).abs() <= 2 * (width + 2) * R.U * size).all()


def test_split_products_captured(ops):
    """A graph with a split forward and dx, replayed on new values between eager calls of other sizes."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w, dy = _make(g, F32, 60, 2560).requires_grad_(True), _make(g, F32, 2560, 2560, std=0.02), _make(g, F32, 60, 2560)

    def step():
        y = ops.linear_act(x, w, activation="gelu")
        return [y.detach(), torch.autograd.grad(y, x, dy)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(3):
        with torch.no_grad():
            x.mul_(-0.5)
        want = step()
        ops.linear_act(x[:7].detach(), w)
        for o in outs:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), f"turn {turn}"


@pytest.mark.parametrize("t", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("case", F.NORM, ids=str)
def test_norm_forms(ops, t, case):
    T.test_norm_gate_and_its_gradients(ops, t, *case)
