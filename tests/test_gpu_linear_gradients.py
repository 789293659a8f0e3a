"""GPU tests of what the linear layer keeps for its backward and what its gradients make of it."""
import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import protein_clip_amd  # noqa: F401
    from protein_clip_amd import _lib, ops as _ops
    assert _lib.load().pclip_check_device(0) == 0, _lib.load().pclip_last_error()
    return _ops


def slope_error(z, slope, t):
    """Relative precision everywhere: exp(-z^2 / 2) and exp(z) turn the argument's roundings (four, of z^2 / 2 or z) into relative ones,
    the fitted tail and the hardware's exp and reciprocal bring 4e-6; near the zero of gelu's slope (z = -0.75) and silu's (z = -1.28) two terms
    of at most 0.3 cancel.  bfloat16 keeps the slope as a float of 11 bits, down to 2^-40."""
    relative = 4e-6 + (z * z / 2 + z.abs()) * 4 * R.U
    err = slope.abs() * relative + torch.where(z.abs() < 3, 4e-6, 0.0)
    return err + (R.half(F16) * slope.abs() + 2.0 ** -40 if t == BF16 else 0.0)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("name", ["gelu", "silu"])
def test_slopes_of_saturated_units(ops, t, name):
    """One unit of one input, so that the gradient is the slope: as exact, relatively, far from zero as near it."""
    low = -6.5 if name == "gelu" else -14.0   # gelu's slope there is 1.7e-9, silu's 1.1e-5
    z = torch.cat([torch.linspace(low, -3.0, 300), torch.linspace(-3.0, 8.0, 100)]).to(t)
    x = z[:, None].cuda().requires_grad_(True)
    y = ops.linear_act(x, torch.ones(1, 1, dtype=t, device="cuda"), activation=name)
    dy = torch.ones_like(y)
    y.backward(dy)
    z = z.double()
    slope = R.act(z, name)[1]
    R.assert_within(x.grad[:, 0], slope, R.rounded(slope, slope_error(z, slope, t), t), "dx")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("name,centre", [("gelu", -4.5), ("gelu", -6.0), ("silu", -12.0), ("silu", -15.0)])
@pytest.mark.parametrize("res", [False, True])
def test_gradients_of_a_layer_of_saturated_units(ops, t, name, centre, res):
    """Every unit's input lies around ``centre``: dx, dW and db still have the precision of their type."""
    g = torch.Generator().manual_seed(7)
    M, K, N = 200, 24, 40
    x, w = (torch.randn(M, K, generator=g) * 0.5).to(t), (torch.randn(N, K, generator=g) * 0.2).to(t)
    b, dy = torch.full((N,), centre).to(t), (torch.randn(M, N, generator=g) * 64).to(t)
    xw, ww, bw, dw = (v.double() for v in (x, w, b, dy))
    z = xw @ ww.t() + bw
    ez = (K + 1) * R.U * (xw.abs() @ ww.abs().t() + bw.abs())
    slope = R.act(z, name)[1]
    es = slope_error(z, slope, t) + slope.abs() * (z.abs() + 2) * ez   # the logarithm of the slope changes by |z| + 1 / |z| at most
    dz = dw * slope
    edz = dw.abs() * es
    rounded_dz = R.rounded(dz, edz, t)
    sums = lambda value, err, size, n: (value, R.rounded(value, err + (n + 8) * R.U * (size + err), t))
    leaves = [v.cuda().requires_grad_(True) for v in (x, w, b)]
    y = ops.linear_act(*leaves, torch.zeros(M, N, dtype=t, device="cuda") if res else None, activation=name)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    R.assert_within(grads[0], *sums(dz @ ww, rounded_dz @ ww.abs(), dz.abs() @ ww.abs(), N), "dx")
    R.assert_within(grads[1], *sums(dz.t() @ xw, rounded_dz.t() @ xw.abs(), dz.abs().t() @ xw.abs(), M), "dW")
    R.assert_within(grads[2], *sums(dz.sum(0), edz.sum(0), dz.abs().sum(0), M), "db")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("res", [False, True])
def test_nan_reaches_the_gradients(ops, t, name, res):
    """A NaN row of the weight makes its unit's outputs NaN; its gradients are torch's: NaN where the slope is computed from the value,
    dy where ReLU passes it on.  The other units stay finite."""
    g = torch.Generator().manual_seed(9)
    M, K, N = 90, 24, 33
    x, w, b, dy = (torch.randn(*s, generator=g).to(t) for s in ((M, K), (N, K), (N,), (M, N)))
    w[5] = float("nan")
    plain = [v.double().requires_grad_(True) for v in (x, w, b)]
    z = plain[0] @ plain[1].t() + plain[2]
    act = {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[name]
    want = torch.autograd.grad(act(z), plain, dy.double())
    leaves = [v.cuda().requires_grad_(True) for v in (x, w, b)]
    y = ops.linear_act(*leaves, torch.ones(M, N, dtype=t, device="cuda") if res else None, activation=name)
    assert y[:, 5].isnan().all() and torch.isfinite(y[:, :5]).all() and torch.isfinite(y[:, 6:]).all()
    for got, ref, what in zip(torch.autograd.grad(y, leaves, dy.cuda()), want, ("dx", "dW", "db")):
        got = got.double().cpu()
        assert torch.equal(got.isnan(), ref.isnan()), what
        fine = ~ref.isnan()
        # 90 products or fewer of values of order one, those of dz rounded: six half steps of the type and 2^-23 a term of the sum of sizes
        tol = 6 * R.half(t) * (1 + ref[fine].abs()) * 10 + 128 * R.U * 100
        assert ((got[fine] - ref[fine]).abs() <= tol).all(), what




def test_relu_outputs_too_small_for_their_type(ops):
    """float16 rounds values up to 2^-25 to zero.  Their slope is one all the same; that of zero and of negative values is zero."""
    scale = torch.tensor([1.0, 0.5, 0.0, -0.5, -1.0, 2.0 ** -10, -(2.0 ** -10)])
    x = (scale[:, None] * 2.0 ** -13).to(F16).cuda().requires_grad_(True)
    w = torch.full((1, 1), 2.0 ** -13, dtype=F16, device="cuda", requires_grad=True)
    b = torch.zeros(1, dtype=F16, device="cuda", requires_grad=True)
    y = ops.linear_act(x, w, b, activation="relu")
    assert not y.any()
    y.backward(torch.full_like(y, 512.0))
    kept = (scale > 0).double()
    assert torch.equal(x.grad[:, 0].double().cpu(), kept * 2.0 ** -4)
    assert b.grad.item() == 512 * kept.sum().item()
    # the sum of three products of 512 and x's own values, rounded once
    want = 512 * (x.detach()[:, 0].double().cpu() * kept).sum()
    assert abs(w.grad.item() - want.item()) <= R.half(F16) * want.item()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,width,out", [(1, 8, 3), (37, 24, 40), (64, 16, 16), (65, 7, 5), (5000, 40, 136), (20000, 8, 600)])
@pytest.mark.parametrize("name", ["none", "relu", "gelu"])
def test_gradients_of_some_operands_only(ops, t, rows, width, out, name):
    """The bias alone, with the input, with the weight: each as when all are wanted."""
    g = torch.Generator().manual_seed(rows)
    x, w, b, dy = ((torch.randn(*s, generator=g) * f).to(t) for s, f in (((rows, width), 1.0), ((out, width), width ** -0.5), ((out,), 1.0), ((rows, out), 1.0)))
    want = R.linear_bounds(x.double(), w.double(), b.double(), None, dy.double(), name, t)
    for mask in (4, 5, 6, 1, 2):
        leaves = [v.cuda().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((x, w, b))]
        y = ops.linear_act(*leaves, activation=name)
        wanted = [v for v in leaves if v.requires_grad]
        names = [n for v, n in zip(leaves, ("x", "weight", "bias")) if v.requires_grad]
        for got, n in zip(torch.autograd.grad(y, wanted, dy.cuda()), names):
            R.assert_within(got, *want[n], f"{mask}: {n}")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "relu", "silu"])
def test_wanted_gradients_whatever_operands_are_given(ops, t, name):
    """The wrapper of the kernels with every choice of wanted gradients, with all operands and with those that the choice needs."""
    from protein_clip_amd import kernels as K
    g = torch.Generator(device="cuda").manual_seed(4)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)
    x, w, b, dy = make(700, 72), make(56, 72), make(56), make(700, 56)
    y, slope = K.linear_fwd(x, w, b, None, name, name == "silu")
    saved = {"none": (None, False), "relu": (y, True), "silu": (slope, False)}[name]
    full = K.linear_bwd(x, w, dy, *saved, name)
    for mask in range(1, 8):
        want = [bool(mask >> i & 1) for i in range(3)]
        for got in (K.linear_bwd(x, w, dy, *saved, name, *want), K.linear_bwd(x if want[1] else None, w if want[0] else None, dy, *saved, name, *want)):
            for i in range(3):
                if not want[i]:
                    assert got[i] is None
                elif i < 2:
                    assert torch.equal(got[i], full[i])
                else:   # the column sum alone, or with the weight's product: the same 700 terms in another order, each sum rounded once
                    size = dy.double().abs().sum(0) * 1.13
                    assert ((got[i].double() - full[i].double()).abs() <= 2 * 708 * R.U * size + 2 * R.half(t) * full[i].double().abs()).all()
