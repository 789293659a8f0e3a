"""GPU tests of the token-head operators (linear layer with its epilogue, norms around a block, gradient clipping) through
``protein_clip_amd.ops``, against plain 64-bit forms, at the sizes and layouts where they can go wrong."""
import math

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


def make(g, t, *shape, std=1.0, mean=0.0):
    """A CPU tensor of type t (its values are what both sides see)."""
    return (torch.randn(*shape, generator=g) * std + mean).to(t)


def leaf(t):
    return None if t is None else t.cuda().requires_grad_(True)


def wide(t):
    return None if t is None else t.double()


# ---- linear --------------------------------------------------------------------------------------------
LINEAR = [   # rows, width, out: single elements, one token, odd everything, both sides of every tile and step, many rows
    (1, 1, 1, "none", True, False), (1, 640, 128, "relu", True, False), (3, 8, 5, "gelu", True, True), (31, 640, 128, "none", True, False),
    (16, 7, 64, "silu", False, False), (63, 65, 129, "relu", True, True), (64, 64, 64, "gelu", False, False), (130, 637, 331, "silu", True, True),
    (129, 129, 257, "gelu", True, False), (300, 320, 200, "relu", False, False), (2000, 16, 24, "none", True, True), (2047, 33, 17, "relu", True, False),
    (513, 1280, 96, "gelu", True, True), (4100, 128, 128, "relu", True, False), (260, 72, 2560, "none", False, True),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,width,out,name,has_bias,has_res", LINEAR)
def test_linear_and_its_gradients(ops, t, rows, width, out, name, has_bias, has_res):
    g = torch.Generator().manual_seed(rows * 7 + width)
    x, w = make(g, t, rows, width), make(g, t, out, width, std=width ** -0.5)
    b = make(g, t, out, std=0.3) if has_bias else None
    r = make(g, t, rows, out) if has_res else None
    dy = make(g, t, rows, out)
    want = R.linear_bounds(wide(x), wide(w), wide(b), wide(r), wide(dy), name, t)
    xs, ws, bs, rs = leaf(x), leaf(w), leaf(b), leaf(r)
    y = ops.linear_act(xs, ws, bs, rs, activation=name)
    with torch.no_grad():
        R.assert_within(ops.linear_act(xs, ws, bs, rs, activation=name), *want["y"], "y without a graph")
    R.assert_within(y, *want["y"], "y")
    y.backward(dy.cuda())
    R.assert_within(xs.grad, *want["x"], "dx")
    R.assert_within(ws.grad, *want["weight"], "dW")
    if has_bias:
        R.assert_within(bs.grad, *want["bias"], "db")
    if has_res:
        assert torch.equal(rs.grad.cpu(), dy)


def test_linear_same_bits_again(ops):
    """Sums over rows run in a fixed order: two calls agree bit for bit."""
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (make(g, BF16, *s).cuda() for s in ((3001, 200), (72, 200), (72,), (3001, 72)))
    runs = []
    for _ in range(2):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        y = ops.linear_act(*leaves, activation="gelu")
        runs.append([y.detach()] + list(torch.autograd.grad(y, leaves, dy)))
    assert all(torch.equal(p, q) for p, q in zip(*runs))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_linear_layouts(ops, t):
    """Leading dimensions, a transposed weight, sliced rows, a base address between two 16-byte steps, broadcast residuals, other operand types."""
    g = torch.Generator().manual_seed(5)
    x, w, b, r = make(g, t, 4, 37, 48), make(g, t, 40, 48, std=0.15), make(g, t, 40), make(g, t, 37, 40)
    dy = make(g, t, 4, 37, 40)
    flat = lambda v: None if v is None else v.double().reshape(-1, v.shape[-1])
    want = R.linear_bounds(flat(x), wide(w), wide(b), flat(r.expand(4, 37, 40)), flat(dy), "silu", t)
    spare = torch.zeros(x.numel() + 1, dtype=t, device="cuda")
    spare[1:] = x.cuda().reshape(-1)
    views = {
        "plain": (x.cuda(), w.cuda(), b.cuda()),
        "odd address": (spare[1:].view(x.shape), w.cuda(), b.cuda()),
        "transposed weight": (x.cuda(), w.cuda().t().contiguous().t(), b.cuda()),
        "sliced rows": (torch.stack([x, x * 2], 2).cuda()[:, :, 0], w.cuda(), torch.stack([b, b], 1).cuda()[:, 0]),
        "32-bit parameters": (x.cuda(), w.float().cuda(), b.float().cuda()),
    }
    for what, (xv, wv, bv) in views.items():
        leaves = [v.detach().requires_grad_(True) for v in (xv, wv, bv, r.cuda())]
        y = ops.linear_act(*leaves, activation="silu")
        assert y.shape == (4, 37, 40)
        R.assert_within(y.reshape(-1, 40), *want["y"], what + ": y")
        grads = torch.autograd.grad(y, leaves, dy.cuda())
        assert [q.dtype for q in grads] == [v.dtype for v in leaves]
        R.assert_within(grads[0].reshape(-1, 48), *want["x"], what + ": dx")
        R.assert_within(grads[1], *want["weight"], what + ": dW")
        R.assert_within(grads[2], *want["bias"], what + ": db")
        total = dy.double().sum(0)
        R.assert_within(grads[3], total, R.rounded(total, 4 * R.half(t) * dy.double().abs().sum(0), t), what + ": dresidual")


def test_linear_only_what_is_wanted(ops):
    """A frozen input, a frozen weight, a frozen bias, each alone; and gradients that arrive expanded from a sum."""
    g = torch.Generator().manual_seed(8)
    x, w, b = make(g, F32, 50, 24), make(g, F32, 12, 24), make(g, F32, 12)
    want = R.linear_bounds(wide(x), wide(w), wide(b), None, torch.ones(50, 12, dtype=torch.float64), "gelu", F32)
    for mask in range(1, 8):
        leaves = [v.cuda().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((x, w, b))]
        ops.linear_act(*leaves, activation="gelu").sum().backward()
        for v, n in zip(leaves, ("x", "weight", "bias")):
            if v.requires_grad:
                R.assert_within(v.grad, *want[n], n)
            else:
                assert v.grad is None


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_linear_no_rows(ops, t):
    x, w, b = (torch.ones(*s, dtype=t, device="cuda", requires_grad=True) for s in ((2, 0, 8), (4, 8), (4,)))
    y = ops.linear_act(x, w, b, activation="relu")
    assert y.shape == (2, 0, 4) and y.dtype == t
    y.sum().backward()
    assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
def test_linear_extreme_values(ops, t, name):
    """Activations at the far ends (also where z itself is infinite), and a NaN row that stays in its row."""
    big = 60000.0 if t == F16 else 1e30
    z = torch.tensor([-big, -100.0, -20.0, -5.0, -1.0, 0.0, 1.0, 5.0, 20.0, 100.0, big])
    x = z.to(t)[:, None].cuda().requires_grad_(True)
    w = torch.ones(1, 1, dtype=t, device="cuda")
    y = ops.linear_act(x, w, activation=name)
    y.backward(torch.ones_like(y))
    value, slope = R.act(z.to(t).double(), name)
    tol = 8e-6 + 2 * R.half(t)
    R.assert_within(y[:, 0], value, tol * value.abs() + 1e-6, "y")
    R.assert_within(x.grad[:, 0], slope, 2 * tol + 0 * slope, "slope")
    rows = torch.ones(70, 40, dtype=t)
    rows[3] = float("nan")
    rows[5, 2] = float("inf")
    out = ops.linear_act(rows.cuda(), torch.ones(33, 40, dtype=t, device="cuda"), activation=name)
    ok = torch.ones(70, dtype=torch.bool)
    ok[[3, 5]] = False
    assert torch.isfinite(out[ok.cuda()]).all() and out[3].isnan().all() and (out[5] == float("inf")).all()


# ---- norms around a block -----------------------------------------------------------------------------------
NORM = [   # batch, tokens, width, gate, after, before, kind, residual, scale
    (1, 1, 640, "none", None, "affine", "layer", True, 1.0), (2, 3, 8, "element", "affine", "affine", "rms", True, 0.5),
    (1, 5, 1, "channel", "affine", "plain", "layer", True, 1.0), (3, 70, 128, "keep", "affine", None, "layer", False, 1 / 0.9),
    (4, 33, 127, "sequence", "affine", "affine", "layer", True, 0.25), (5, 9, 129, "channel", "plain", "affine", "rms", True, 1.0),
    (2, 40, 257, "element", None, "plain", "layer", True, 2.0), (7, 300, 64, "sequence", "affine", None, "rms", False, 1.0),
    (700, 2, 96, "sequence", "affine", "affine", "rms", True, 1.0), (2, 60, 640, "sequence", "affine", "affine", "rms", True, 0.5),
    (3, 11, 1025, "channel", "affine", "affine", "layer", True, 0.25), (2, 9, 4096, "keep", "plain", "affine", "layer", True, 1.0),
    (1, 7, 2049, "sequence", "affine", "affine", "layer", False, 1.0), (2, 5, 513, "none", None, None, "layer", True, 0.5),
    (1, 3000, 24, "channel", "affine", "affine", "rms", True, 1.0),
]


def _norm_operands(g, t, batch, tokens, width, gate, after, before, kind, res, ptype):
    u = make(g, t, batch, tokens, width, std=1.5, mean=0.5)
    r = make(g, t, batch, tokens, width, std=2.0) if res else None
    shapes = {"channel": (width,), "sequence": (batch, 1, width), "element": (batch, tokens, width)}
    gt = None
    if gate == "keep":
        gt = (torch.rand(batch, tokens, width, generator=g) >= 0.3)
    elif gate != "none":
        gt = make(g, t, *shapes[gate], std=0.5, mean=0.5)
    pair = lambda how: None if how is None else (None, None) if how == "plain" else (
        make(g, ptype, width, std=0.2, mean=1.0), make(g, ptype, width, std=0.2) if kind == "layer" else None)
    return u, r, gt, pair(after), pair(before)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("batch,tokens,width,gate,after,before,kind,res,scale", NORM)
def test_norm_gate_and_its_gradients(ops, t, batch, tokens, width, gate, after, before, kind, res, scale):
    g = torch.Generator().manual_seed(batch * 31 + width)
    ptype = t if width % 2 else F32
    u, r, gt, pa, pb = _norm_operands(g, t, batch, tokens, width, gate, after, before, kind, res, ptype)
    dy, dn = make(g, t, batch, tokens, width), make(g, t, batch, tokens, width) if before else None
    pw = lambda pair: None if pair is None else tuple(wide(p) for p in pair)
    scale32 = torch.tensor(scale).double().item()
    want = R.norm_gate_bounds(wide(u), wide(r), wide(gt), scale32, pw(pa), pw(pb), kind, wide(dy), wide(dn), t)
    us, rs = leaf(u), leaf(r)
    gs = gt.cuda() if gate == "keep" else leaf(gt)
    las, lbs = (None if pair is None else tuple(leaf(p) for p in pair) for pair in (pa, pb))
    call = lambda: ops.norm_gate_residual(us, rs, gs, scale=scale, after=las, before=lbs, norm=kind)
    outs = call()
    outs = outs if before else (outs,)
    with torch.no_grad():
        plain = call()
        assert all(torch.equal(p, q) for p, q in zip(plain if before else (plain,), outs))
    for o, n in zip(outs, ("y", "n")):
        R.assert_within(o, *want[n], n)
    torch.autograd.backward(outs, [v.cuda() for v in (dy, dn) if v is not None])
    R.assert_within(us.grad, *want["u"], "du")
    if res:
        R.assert_within(rs.grad, *want["residual"], "dresidual")
    if gate in ("channel", "sequence", "element"):
        value, err = want["gate"]
        if gate == "element":
            R.assert_within(gs.grad, value, R.rounded(value, err, t), "dgate")
        else:
            s, tol = R.column_sum(value, err, t, batch * tokens if gate == "channel" else tokens, (0, 1) if gate == "channel" else 1)
            R.assert_within(gs.grad.reshape(s.shape), s, tol, "dgate")
    for pair, names in ((las, ("wa", "ba")), (lbs, ("wb", "bb"))):
        for p, n in zip(pair or (), names):
            if p is not None:
                R.assert_within(p.grad, *R.column_sum(*want[n], ptype, batch * tokens, (0, 1)), "d" + n)


def test_norm_gate_broadcasts_and_partial_gradients(ops):
    """Gates of other broadcast patterns, a residual that is broadcast, a gradient that reaches one output only, frozen operands."""
    g = torch.Generator().manual_seed(4)
    u, gt, r = make(g, F32, 3, 5, 2, 24), make(g, F32, 1, 5, 1, 24), make(g, F32, 2, 24)
    w = make(g, F32, 24)
    for use in ("y", "n", "both"):
        cpu = [v.double().requires_grad_(True) for v in (u, r, gt, w)]
        gpu = [leaf(v) for v in (u, r, gt, w)]
        for leaves, fn in ((cpu, lambda a, b, c, d: R.norm_gate(a, b, c, 0.5, (d, None), (None, None), "layer")),
                           (gpu, lambda a, b, c, d: ops.norm_gate_residual(a, b, c, scale=0.5, after=(d, None), before=(None, None)))):
            y, n = fn(*leaves)
            dy, dn = torch.cos(torch.arange(y.numel())).reshape(y.shape).to(y), torch.sin(torch.arange(y.numel()) * 0.7).reshape(y.shape).to(y)
            ((y * dy).sum() * (use != "n") + (n * dn).sum() * (use != "y")).backward() if use == "both" else ((y * dy) if use == "y" else (n * dn)).sum().backward()
        for p, q, what in zip(gpu, cpu, ("u", "residual", "gate", "weight")):
            # f32 throughout, values of order one, sums over at most 30 rows: 2^-23 * 64 roundings * 30
            R.assert_within(p.grad, q.grad, 64 * 30 * R.U * (1 + q.grad.abs()), f"{use}: {what}")
    frozen = ops.norm_gate_residual(u.cuda(), gate=leaf(gt), after=(w.cuda(), None))
    frozen.sum().backward()   # only the gate takes a gradient


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_norm_gate_rows_that_are_alike(ops, t):
    """A constant row has no spread: the norm returns its bias, gradients stay finite; a NaN row stays in its row; no rows at all."""
    u = torch.full((4, 40), 3.0, dtype=t)
    u[1] = 0
    u[2, 7] = float("nan")
    b = torch.linspace(-1, 1, 40)
    ub = u.cuda().requires_grad_(True)
    wb = torch.ones(40, device="cuda", requires_grad=True)
    y = ops.norm_gate_residual(ub, after=(wb, b.cuda()))
    assert y[2].isnan().all()
    for i in (0, 1, 3):
        R.assert_within(y[i], b.double(), R.rounded(b.double(), 1e-3 * torch.ones(40), t), "constant row")   # 3 - mean is off by 2 steps of f32, times 1 / sqrt(eps) = 316
    grads, = torch.autograd.grad(y[[0, 1, 3]].sum(), ub)
    assert torch.isfinite(grads[[0, 1, 3]]).all()
    e = torch.empty(3, 0, 40, dtype=t, device="cuda", requires_grad=True)
    y, n = ops.norm_gate_residual(e, e, before=(wb, None))
    (y.sum() + n.sum()).backward()
    assert y.shape == n.shape == e.grad.shape == e.shape and not wb.grad.any()


# ---- gradient norm and clipping --------------------------------------------------------------------------------
def _many(g, t, count):
    sizes = [(1,), (7,), (128, 640), (128,), (3, 5, 7), (8192,), (8193,), (16385,), (0,), (33, 33)]
    return [make(g, t, *sizes[i % len(sizes)], std=0.1 + i % 3) for i in range(count)]


@pytest.mark.parametrize("count", [1, 2, 29, 120, 121, 300])
@pytest.mark.parametrize("t", TYPES, ids=str)
def test_clip_norm_and_values(ops, t, count):
    g = torch.Generator().manual_seed(count)
    grads = _many(g, t, count)
    exact = math.sqrt(math.fsum(float((v.double() ** 2).sum()) for v in grads))
    for limit in (0.25 * exact, 4 * exact + 1):
        dev = [v.cuda() for v in grads]
        before = [v.clone() for v in dev]
        norm = ops.clip_grads(dev, limit)
        # f64 squares and sums, one rounding to f32; the factor: an addition, a division; the product
        assert abs(norm.item() - exact) <= 2.0 ** -23 * exact
        factor = min(1.0, limit / (exact + 1e-6))
        for v, got, was in zip(grads, dev, before):
            if factor == 1.0:
                assert torch.equal(got, was)
            else:
                ref = v.double() * factor
                R.assert_within(got, ref, R.rounded(ref, 6 * R.U * ref.abs(), t), "clipped")
        assert torch.equal(ops.grad_norm(before), norm) and torch.equal(ops.grad_norm(before), norm)


@pytest.mark.parametrize("s", TYPES, ids=str)
@pytest.mark.parametrize("t", TYPES, ids=str)
def test_clip_into_other_types(ops, s, t):
    """A reduced buffer of one type into gradients of another, as views of flat buffers at odd places."""
    g = torch.Generator().manual_seed(1)
    src = _many(g, s, 14)
    sizes = [v.numel() for v in src]
    for lead in (0, 1):
        flat_s = torch.zeros(sum(sizes) + lead, dtype=s, device="cuda")
        flat_t = torch.full((sum(sizes) + 3,), 7.0, dtype=t, device="cuda")
        flat_s[lead:] = torch.cat([v.reshape(-1) for v in src]).cuda()
        a = [v.view(q.shape) for v, q in zip(flat_s[lead:].split(sizes), src)]
        b = [v.view(q.shape) for v, q in zip(flat_t[1:-2].split(sizes), src)]
        norm = ops.clip_grads(a, 2.0, out=b)
        factor = 2.0 / (norm.double().item() + 1e-6)
        for v, got in zip(src, b):
            ref = v.double() * factor
            R.assert_within(got, ref, R.rounded(ref, 6 * R.U * ref.abs(), t), "clipped")
        assert flat_t[0] == 7 and (flat_t[-2:] == 7).all()


def test_clip_extreme_values(ops):
    big = [torch.full((5000,), 1e30, device="cuda"), torch.full((10,), 1e-30, device="cuda")]
    assert abs(ops.grad_norm(big).item() / (1e30 * math.sqrt(5000)) - 1) < 1e-6
    tiny = [torch.full((4096,), 1e-30, device="cuda")]
    assert abs(ops.grad_norm(tiny).item() / 6.4e-29 - 1) < 1e-6
    for bad in (float("inf"), float("nan")):
        v = [torch.tensor([1.0, bad, 2.0], device="cuda"), torch.ones(9, device="cuda")]
        norm = ops.clip_grads(v, 1.0)
        if bad != bad:
            assert norm.isnan() and v[0].isnan().all() and v[1].isnan().all()
        else:
            assert norm.isinf() and v[0][1].isnan() and not v[1].any() and v[0][0] == 0
    zero = [torch.zeros(100, device="cuda")]
    assert ops.clip_grads(zero, 0.0).item() == 0 and not zero[0].any()
    ones = [torch.ones(100, device="cuda")]
    assert ops.clip_grads(ones, 0.0).item() == 10 and not ones[0].any()
    assert ops.grad_norm([torch.empty(0, device="cuda")]).item() == 0


def test_clip_grad_norm_on_parameters(ops):
    """Against torch's own function, in a transposed layout too; parameters without a gradient are passed over."""
    g = torch.Generator().manual_seed(2)
    ps = [torch.zeros(s, device="cuda", requires_grad=True) for s in ((5, 9), (300,), (4, 4), (1,))]
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    for i, (p, q) in enumerate(zip(ps, qs)):
        if i != 2:
            v = torch.randn(p.shape, generator=g).cuda()
            p.grad = v.t().contiguous().t() if v.dim() == 2 else v.clone()
            q.grad = v.clone()
    norm, ref = ops.clip_grad_norm_(ps, 1.5), torch.nn.utils.clip_grad_norm_(qs, 1.5)
    torch.testing.assert_close(norm, ref, rtol=2e-6, atol=0)
    for p, q in zip(ps, qs):
        if q.grad is not None:
            torch.testing.assert_close(p.grad, q.grad, rtol=2e-6, atol=0)
    assert ops.clip_grad_norm_(ps[2], 1.0).item() == 0
    ps[0].grad[1, 1] = float("inf")
    kept = ps[1].grad.clone()
    with pytest.raises(RuntimeError, match="norm is inf"):
        ops.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.equal(ps[1].grad, kept)


def test_clip_refusals(ops):
    from protein_clip_amd._lib import PclipError
    a = torch.ones(64, device="cuda")
    for bad, what in (([a, a], "share memory"), ([a, a[10:20]], "share memory"), ([a.view(8, 8)[:, :4]], "gaps"), ([torch.ones(1, device="cuda").expand(9)], "gaps"),
                      ([a, torch.ones(3)], "expected a dense"), ([a.double()], "expected a dense"), ([], "no tensors")):
        with pytest.raises(PclipError, match=what):
            ops.clip_grads(bad, 1.0)
    with pytest.raises(PclipError, match="shares memory"):
        ops.clip_grads([a[:32]], 1.0, out=[a[16:48]])
    with pytest.raises(PclipError, match="destinations"):
        ops.clip_grads([a], 1.0, out=[])
    with pytest.raises(PclipError, match="shapes"):
        ops.clip_grads([a], 1.0, out=[torch.ones(63, device="cuda")])
    with pytest.raises(PclipError, match="destination 0"):
        ops.clip_grads([a.view(8, 8)], 1.0, out=[torch.ones(8, 8, device="cuda").t()])
    with pytest.raises(PclipError, match="destination 0"):
        ops.clip_grads([a], 1.0, out=[torch.ones(64, device="cuda").double()])
    with pytest.raises(PclipError, match="tensor 0"):
        ops.clip_grads([torch.eye(3, device="cuda").to_sparse()], 1.0)
    for limit in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_grads([a], limit)
    assert ops.grad_norm([a, a]).item() == pytest.approx(math.sqrt(128))   # reading one tensor twice is no conflict
    assert torch.equal(a, torch.ones(64, device="cuda"))


# ---- streams, graphs, together ----------------------------------------------------------------------------------
def _token_step(ops, x, p, keep, grads=None):
    """Projection, one Linear-ReLU-norm-dropout block, last layer, a residual join with the next norm; gradients, then clipping."""
    h = ops.linear_act(x, p["w0"], p["b0"])
    a = ops.linear_act(h, p["w1"], p["b1"], activation="relu")
    a = ops.norm_gate_residual(a, gate=keep, scale=1 / 0.9, after=(p["g1"], p["c1"]))
    o = ops.linear_act(a, p["w2"], p["b2"], residual=h, activation="gelu")
    y, n = ops.norm_gate_residual(o, h, p["gate"], scale=0.5, after=(p["g1"], None), before=(p["g2"], p["c2"]))
    loss = (y.float() * n.float()).mean() + y.float().square().mean()
    names = list(p)
    out = list(torch.autograd.grad(loss, [p[k] for k in names]))
    norm = ops.clip_grads(out, 0.05)
    return [loss.detach(), norm] + out


def _token_params(t, width=96, d=64, out_device="cuda"):
    g = torch.Generator().manual_seed(12)
    p = {"w0": make(g, t, d, width, std=0.1), "b0": make(g, t, d), "w1": make(g, t, d, d, std=0.12), "b1": make(g, t, d), "g1": make(g, F32, d, mean=1.0, std=0.1),
         "c1": make(g, F32, d, std=0.1), "w2": make(g, t, d, d, std=0.12), "b2": make(g, t, d), "gate": make(g, t, d, mean=0.5), "g2": make(g, F32, d, mean=1.0, std=0.1),
         "c2": make(g, F32, d)}
    x = make(g, t, 6, 50, width)
    keep = torch.rand(6, 50, d, generator=g) >= 0.1
    return x, p, keep


def test_a_step_of_all_operators_together(ops):
    """The operators in a row, as a tower's token head uses them, in f32 against the same composition in 64 bits (every
    intermediate of order one, some forty operations deep: 2^-23 * 4096 of the largest gradient)."""
    x, p, keep = _token_params(F32)
    got = _token_step(ops, x.cuda(), {k: leaf(v) for k, v in p.items()}, keep.cuda())

    class Plain:
        linear_act = staticmethod(lambda x, w, b, residual=None, activation="none": R.linear(x.reshape(-1, x.shape[-1]), w, b, None, activation).reshape(
            x.shape[:-1] + (w.shape[0],)) + (0 if residual is None else residual))

        @staticmethod
        def norm_gate_residual(u, r=None, gate=None, scale=1.0, after=None, before=None):
            out = R.norm_gate(u, r, gate, scale, after, before, "layer")
            return out if before else out[0]

        @staticmethod
        def clip_grads(v, limit):
            norm = torch.sqrt(sum((q ** 2).sum() for q in v))
            for q in v:
                q.mul_(min(1.0, limit / (norm.item() + 1e-6)))
            return norm

    class Widen(dict):
        pass

    want = None
    p64 = {k: v.double().requires_grad_(True) for k, v in p.items()}
    orig_float = torch.Tensor.float
    try:
        torch.Tensor.float = lambda self: self   # the 64-bit side stays in 64 bits
        want = _token_step(Plain, x.double(), p64, keep.double())
    finally:
        torch.Tensor.float = orig_float
    for a, b, what in zip(got, want, ["loss", "norm"] + list(p)):
        R.assert_within(a, b.detach(), 4096 * R.U * (b.detach().abs().max() + 0 * b.detach()), what)


def test_on_another_stream(ops):
    """The whole step on a side stream gives what the default stream gives, bit for bit."""
    x, p, keep = _token_params(BF16)
    xs, ks = x.cuda(), keep.cuda()
    want = _token_step(ops, xs, {k: leaf(v) for k, v in p.items()}, ks)
    ps = {k: leaf(v) for k, v in p.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _token_step(ops, xs, ps, ks)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_captured_graphs_replayed_in_turn(ops):
    """Two graphs of the step on inputs of their own, replayed in turn with eager work between: each replay equals the eager result."""
    graphs = []
    for seed in (0, 1):
        x, p, keep = _token_params(BF16)
        xs, ks = (x * (1 + seed)).cuda(), keep.cuda()
        ps = {k: leaf(v) for k, v in p.items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _token_step(ops, xs, ps, ks)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _token_step(ops, xs, ps, ks)
        graphs.append((graph, outs, xs, ps, ks))
    for turn in range(3):
        for graph, outs, xs, ps, ks in graphs:
            xs.mul_(0.5)
            eager = _token_step(ops, xs, ps, ks)
            for o in outs:
                o.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), f"turn {turn}"


def test_gradients_against_differences(ops):
    """Directional differences of the f32 forward against its gradients.  Step 2^-6 along a direction of length one: the third-order
    term is below 2^-12 of the gradient's size, the forward's rounding (2^-23 * 100 terms of order one over 2^-5) below 2^-11."""
    g = torch.Generator().manual_seed(21)
    d = 24
    base = {"x": make(g, F32, 6, d), "w": make(g, F32, d, d, std=0.2), "b": make(g, F32, d), "r": make(g, F32, 6, d), "gate": make(g, F32, d), "wa": make(g, F32, d, mean=1.0)}
    cot = make(g, F32, 2, 6, d).cuda()

    def value(v):
        a = ops.linear_act(v["x"], v["w"], v["b"], v["r"], activation="gelu")
        y, n = ops.norm_gate_residual(a, v["r"], v["gate"], scale=0.7, after=(v["wa"], None), before=(v["wa"], v["b"]), norm="rms")
        return ((torch.stack([y, n]) * cot).double()).sum()

    leaves = {k: leaf(v) for k, v in base.items()}
    grads = dict(zip(leaves, torch.autograd.grad(value(leaves), list(leaves.values()))))
    for k in base:
        way = make(g, F32, *base[k].shape).cuda()
        way /= way.norm()
        h = 2.0 ** -6
        with torch.no_grad():
            shift = lambda s: value({n: (v + s * way if n == k else v) for n, v in leaves.items()})
            diff = (shift(h) - shift(-h)).item() / (2 * h)
        exact = (grads[k].double() * way.double()).sum().item()
        assert abs(diff - exact) <= 2.0 ** -8 * (1 + grads[k].norm().item()), k


# ---- calls at the edges of what is allowed -------------------------------------------------------------------------
def test_clip_of_many_tensors_captured(ops):
    """A table of more tensors than the kernels' arguments hold, written anew by every replay: replays on new values, with eager
    calls of another table between them, equal the eager results."""
    g = torch.Generator().manual_seed(31)
    src = [make(g, BF16, 1 + 37 * (k % 11)).cuda() for k in range(250)]
    other = [make(g, F32, 5 + k % 7).cuda() for k in range(200)]
    dst = [torch.empty(v.shape, device="cuda") for v in src]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.clip_grads(src, 0.5, out=dst)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(src, 0.5, out=dst)
    for turn in range(3):
        for v in src:
            v.mul_(-0.75)
        want = [torch.empty_like(d) for d in dst]
        want_norm = ops.clip_grads(src, 0.5, out=want)
        ops.clip_grads(other, 0.5)
        for d in dst:
            d.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want_norm) and all(torch.equal(a, b) for a, b in zip(dst, want)), f"turn {turn}"


def test_two_threads_on_two_streams(ops):
    """Two threads run the step on inputs and streams of their own at once; each result equals the one computed alone."""
    import threading
    cases = []
    for k in range(2):
        x, p, keep = _token_params(BF16)
        x = (x * (1 + k)).cuda()
        keep = keep.cuda()
        alone = _token_step(ops, x, {n: leaf(v) for n, v in p.items()}, keep)
        cases.append((x, {n: leaf(v) for n, v in p.items()}, keep, alone))
    torch.cuda.synchronize()
    results = [None, None]

    def work(k):
        x, p, keep, _ = cases[k]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [_token_step(ops, x, p, keep) for _ in range(5)]
        stream.synchronize()
        results[k] = outs

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for k in range(2):
        assert results[k] is not None, f"thread {k} ended early"
        for outs in results[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, cases[k][3])), f"thread {k}"


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("width", [16, 128, 640, 1280, 2560])
def test_norm_gate_at_odd_addresses(ops, t, width):
    """Operands that begin one element (a mask: one byte) behind an aligned address."""
    g = torch.Generator().manual_seed(width)
    rows = 37
    u, r, el, dy, dn = (make(g, t, rows, width) for _ in range(5))
    keep = torch.rand(rows, width, generator=g) >= 0.2

    def shifted(v):
        flat = torch.zeros(v.numel() + 1, dtype=v.dtype, device="cuda")
        flat[1:] = v.cuda().reshape(-1)
        return flat[1:].view(v.shape)

    for gate in (el, keep):
        want = R.norm_gate_bounds(wide(u), wide(r), wide(gate), 0.75, (None, None), (None, None), "layer", wide(dy), wide(dn), t)
        a, b, gt = shifted(u).requires_grad_(True), shifted(r).requires_grad_(True), shifted(gate)
        if gate is el:
            gt.requires_grad_(True)
        y, n = ops.norm_gate_residual(a, b, gt, scale=0.75, after=(None, None), before=(None, None))
        R.assert_within(y, *want["y"], "y")
        R.assert_within(n, *want["n"], "n")
        torch.autograd.backward((y, n), (shifted(dy), shifted(dn)))
        R.assert_within(a.grad, *want["u"], "du")
        R.assert_within(b.grad, *want["residual"], "dresidual")
        if gate is el:
            R.assert_within(gt.grad, want["gate"][0], R.rounded(*want["gate"], t), "dgate")


def test_byte_mask_keeps_what_is_not_zero(ops):
    u = torch.arange(1.0, 9.0, device="cuda").view(2, 4)
    gate = torch.tensor([[0, 1, 2, 255], [128, 0, 0, 3]], dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.norm_gate_residual(u, gate=gate, scale=2.0), torch.where(gate != 0, 2 * u, 0 * u))


def test_one_tensor_in_two_places(ops):
    """The same tensor as block output, residual and gate, and as the input and the residual of a layer: its gradients add up."""
    g = torch.Generator().manual_seed(3)
    v, w, dy = make(g, F32, 9, 24), make(g, F32, 24, 24, std=0.2), make(g, F32, 9, 24)
    a, b = v.double().requires_grad_(True), leaf(v)
    (R.norm_gate(a, a, a, 0.5, (None, None), None, "layer")[0] * dy.double()).sum().backward()
    (ops.norm_gate_residual(b, b, b, scale=0.5, after=(None, None)) * dy.cuda()).sum().backward()
    # values of order one to four, some sixty operations, sums over 24 terms
    R.assert_within(b.grad, a.grad, 64 * 24 * R.U * (1 + a.grad.abs()), "norm_gate")
    a, b = v.double().requires_grad_(True), leaf(v)
    (R.linear(a, w.double(), None, a, "silu") * dy.double()).sum().backward()
    (ops.linear_act(b, w.cuda(), residual=b, activation="silu") * dy.cuda()).sum().backward()
    R.assert_within(b.grad, a.grad, 64 * 24 * R.U * (1 + a.grad.abs()), "linear")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,width,out", [(3, 65536, 2), (3, 2, 65536), (1, 65535, 1)])
def test_linear_at_the_widest(ops, t, rows, width, out):
    g = torch.Generator().manual_seed(out)
    x, w, dy = make(g, t, rows, width), make(g, t, out, width, std=1 / math.sqrt(width)), make(g, t, rows, out)
    b = make(g, t, out)
    want = R.linear_bounds(x.double(), w.double(), b.double(), None, dy.double(), "none", t)
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    y = ops.linear_act(xs, ws, bs)
    y.backward(dy.cuda())
    R.assert_within(y, *want["y"], "y")
    for p, n in ((xs, "x"), (ws, "weight"), (bs, "bias")):
        R.assert_within(p.grad, *want[n], "d" + n)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_beyond_the_limits_is_refused(ops, t):
    from protein_clip_amd._lib import PclipError
    z = lambda *s: torch.zeros(*s, dtype=t, device="cuda")
    for x, w in ((z(1, 65537), z(1, 65537)), (z(1, 1), z(65537, 1))):
        with pytest.raises(PclipError, match="widths"):
            ops.linear_act(x, w)
    with pytest.raises(PclipError, match="row width"):
        ops.norm_gate_residual(z(2, 4097), after=(None, None))
