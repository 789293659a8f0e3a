"""CPU tests of the token-head operators' host side: refusals (before anything is launched), how shapes reach the kernels, the towers
with ``token_dtype`` and the loops with ``max_grad_norm`` on the test-only CPU provider, also on two ranks."""
import ctypes
import os
import socket
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from conftest import is_port_clash

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (ROOT, os.path.join(ROOT, "tests")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

import token_ref as R  # noqa: E402


@pytest.fixture()
def provider():
    import token_cpu_provider as P
    from protein_clip_amd import ops
    real = ops._hip_kernels
    ops._hip_kernels = P
    yield P
    ops._hip_kernels = real


# ---- refusals --------------------------------------------------------------------------------------------
def test_c_entry_points_reject_before_launch():
    from protein_clip_amd import _lib
    lib, one, err = _lib.load(), ctypes.c_void_p(64), lambda: lib.pclip_last_error().decode()

    def linear_fwd(x=one, w=one, M=4, K=8, N=8, dtype=1, act=0, y=one):
        return lib.pclip_linear_fwd(x, w, None, None, M, K, N, dtype, act, y, None, None)

    for bad, what in ((dict(x=None), "null pointer"), (dict(y=None), "null pointer"), (dict(M=0), "M=0"), (dict(K=0), "K=0"), (dict(N=65537), "N=65537"),
                      (dict(M=2**31 - 1), "M=2147483647"), (dict(dtype=3), "unknown type"), (dict(act=4), "unknown activation"), (dict(act=-1), "unknown activation")):
        assert linear_fwd(**bad) == -1 and what in err(), bad

    def linear_bwd(x=one, w=one, dy=one, saved=None, is_out=0, act=0, dx=one, dw=one, db=one, ws=one, n=1 << 30):
        return lib.pclip_linear_bwd(x, w, dy, saved, is_out, 4, 8, 8, 1, act, dx, dw, db, ws, n, None)

    for bad, what in ((dict(dy=None), "null pointer"), (dict(w=None), "null pointer"), (dict(x=None), "null pointer"),
                      (dict(x=None, dw=None), "needs x"), (dict(act=2), "saved is needed"), (dict(act=2, saved=one, is_out=1), "only relu"),
                      (dict(act=2, saved=one, n=16), "workspace too small"), (dict(act=2, saved=one, ws=None), "workspace too small"),
                      (dict(ws=ctypes.c_void_p(72)), "16-byte aligned")):
        assert linear_bwd(**bad) == -1 and what in err(), bad
    assert lib.pclip_linear_bwd_workspace_bytes(0, 8, 8, 1, 0) == 0 and lib.pclip_linear_bwd_workspace_bytes(4, 8, 8, 1, 0) == 0
    assert lib.pclip_linear_bwd_workspace_bytes(4, 8, 8, 1, 2) >= 4 * 8 * 2 and lib.pclip_linear_bwd_workspace_bytes(4096, 8, 8, 1, 0) > 8 * 9 * 4

    def norm_fwd(u=one, gate=None, kind=0, gate_rows=1, after=1, before=0, ptype=0, eps=1e-5, rows=6, d=8, dtype=1, y=one, n=None, stats=None):
        return lib.pclip_norm_gate_fwd(u, None, gate, kind, gate_rows, 1.0, after, None, None, before, None, None, ptype, eps, rows, d, dtype, y, n, stats, None)

    for bad, what in ((dict(u=None), "null pointer"), (dict(y=None), "null pointer"), (dict(before=1), "null pointer"), (dict(rows=0), "rows=0"), (dict(d=4097), "d=4097"),
                      (dict(d=0), "d=0"), (dict(dtype=7), "unknown type"), (dict(ptype=2), "affine parameters"), (dict(after=3), "unknown norm"),
                      (dict(kind=1), "gate kind"), (dict(kind=1, gate=one, gate_rows=4), "does not divide"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                      (dict(stats=ctypes.c_void_p(8)), "16-byte aligned")):
        assert norm_fwd(**bad) == -1 and what in err(), bad

    def norm_bwd(kind=0, gate=None, after=1, before=0, stats=one, dy=one, dn=None, dg=None, dwa=None, dwb=None, ws=None, n=0):
        return lib.pclip_norm_gate_bwd(one, None, gate, kind, 1, 1.0, after, None, None, before, None, None, 0, 1e-5, 6, 8, 1, stats, dy, dn, one, None, dg, dwa, None,
                                       dwb, None, ws, n, None)

    for bad, what in ((dict(dy=None), "null pointer"), (dict(stats=None), "statistics"), (dict(dg=one), "no gradient"), (dict(kind=2, gate=one, dg=one), "no gradient"),
                      (dict(dwb=one), "not there"), (dict(dwa=one), "workspace too small"), (dict(dwa=one, ws=one, n=64), "workspace too small")):
        assert norm_bwd(**bad) == -1 and what in err(), bad
    assert lib.pclip_norm_gate_bwd_workspace_bytes(6, 8, 1, 4) == 0

    ptrs, n8, t = (ctypes.c_void_p * 1)(64), (ctypes.c_int64 * 1)(8), (ctypes.c_int * 1)(0)
    t1, t9, neg, big = (ctypes.c_int * 1)(1), (ctypes.c_int * 1)(9), (ctypes.c_int64 * 1)(-1), (ctypes.c_int64 * 1)(1 << 43)

    def clip(src=ptrs, numel=n8, st=t, dst=ptrs, dt=t, n=1, limit=1.0, eps=1e-6, norm=one, ws=one, nb=1 << 20):
        return lib.pclip_grad_clip(src, numel, st, dst, dt, n, limit, eps, norm, ws, nb, None)

    for bad, what in ((dict(src=None), "null pointer"), (dict(norm=None), "null pointer"), (dict(ws=None), "null pointer"), (dict(dt=None), "null pointer"), (dict(n=0), "n=0"),
                      (dict(limit=-1.0), "max_norm"), (dict(limit=float("nan")), "max_norm"), (dict(eps=float("inf")), "eps"), (dict(nb=8), "workspace too small"),
                      (dict(numel=neg), "-1 elements"), (dict(numel=big), "elements"), (dict(st=t9), "unknown type"), (dict(dt=t1), "two types"),
                      (dict(src=(ctypes.c_void_p * 1)()), "null pointer")):
        assert clip(**bad) == -1 and what in err(), bad


def test_operators_reject_cpu_tensors_and_wrong_shapes():
    from protein_clip_amd import ops
    from protein_clip_amd._lib import PclipError
    x, w = torch.ones(3, 8), torch.ones(4, 8)
    for call in (lambda: ops.linear_act(x, w), lambda: ops.norm_gate_residual(x, after=(None, None)), lambda: ops.clip_grads([x], 1.0), lambda: ops.grad_norm([x]),
                 lambda: ops.linear_act(x.double(), w.double())):
        with pytest.raises(PclipError):
            call()
    for call in (lambda: ops.linear_act(x, torch.ones(4, 7)), lambda: ops.linear_act(x, torch.ones(8)), lambda: ops.linear_act(x, w, torch.ones(5)),
                 lambda: ops.linear_act(x, w, activation="tanh"), lambda: ops.linear_act(x, torch.ones(0, 8)), lambda: ops.norm_gate_residual(x, norm="batch"),
                 lambda: ops.norm_gate_residual(x, after=(torch.ones(7), None)), lambda: ops.norm_gate_residual(x, gate=torch.ones(1, 1, 8)),
                 lambda: ops.norm_gate_residual(x, scale=torch.ones(())), lambda: ops.clip_grads([x], -1.0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.linear_act(x, w, residual=torch.ones(2, 4)), lambda: ops.norm_gate_residual(x, torch.ones(2, 8)), lambda: ops.norm_gate_residual(x, gate=torch.ones(2, 8))):
        with pytest.raises(RuntimeError):   # torch's own message of shapes that do not broadcast
            call()


def test_second_derivatives_are_refused(provider):
    from protein_clip_amd import ops
    x, w = torch.ones(3, 8, requires_grad=True), torch.ones(4, 8, requires_grad=True)
    for y in (ops.linear_act(x, w, activation="gelu"), ops.norm_gate_residual(x, after=(None, None))):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


# ---- the formulas, and how shapes reach them ------------------------------------------------------------------
def test_reference_formulas_against_differences():
    """The plain forms that the GPU results are compared with: their slopes and the provider's gradients against differences, in 64 bits."""
    import token_cpu_provider as P
    g = torch.Generator().manual_seed(0)
    z = torch.randn(50, generator=g, dtype=torch.float64) * 3
    for name in ("none", "relu", "gelu", "silu"):
        h = 1e-6
        diff = (R.act(z + h, name)[0] - R.act(z - h, name)[0]) / (2 * h)
        torch.testing.assert_close(R.act(z, name)[1], diff, rtol=1e-7, atol=1e-8)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x, w, b, s: R.linear(x, w, b, s, "gelu"), (r(3, 5), r(4, 5), r(4), r(3, 4)))
    for kind in ("layer", "rms"):
        assert torch.autograd.gradcheck(lambda u, s, gt, w, b: R.norm_gate(u, s, gt, 0.7, (w, b), (w, None), kind), (r(2, 3, 6), r(2, 3, 6), r(2, 1, 6), r(6), r(6)))
        # the bounds' own closed forms of the gradients
        u, s, gt, w, b, dy, dn = (r(2, 3, 6) for _ in range(3)), None, None, r(6), r(6), None, None
        u, s, e = list(u)
        gt = r(2, 1, 6)
        dy, dn = r(2, 3, 6).detach(), r(2, 3, 6).detach()
        y, n = R.norm_gate(u, s, gt, 0.7, (w, b), (w, b), kind)
        grads = torch.autograd.grad((y, n), (u, s, gt), (dy, dn))
        with torch.no_grad():
            want = R.norm_gate_bounds(u, s, gt, 0.7, (w, b), (w, b), kind, dy, dn, torch.float32)
        torch.testing.assert_close(want["u"][0], grads[0])
        torch.testing.assert_close(want["residual"][0], grads[1])
        torch.testing.assert_close(want["gate"][0].sum(1, keepdim=True), grads[2])
    x, w, b = r(7, 5), r(4, 5), r(4)
    y, slope = P.linear_fwd(x, w, b, None, "silu", True)
    dy = torch.randn(7, 4, generator=g, dtype=torch.float64)
    for got, want in zip(P.linear_bwd(x, w, dy, slope, False, "silu"), torch.autograd.grad(y, (x, w, b), dy)):
        torch.testing.assert_close(got, want)


@pytest.mark.parametrize("shape,gate_rows", [((6,), 60), ((1, 1, 6), 60), ((5, 1, 6), 12), ((5, 12, 6), 1), ((1, 12, 6), None), ((5, 12, 1), None), ((), None), ((1, 6), 60)])
def test_gate_patterns(provider, monkeypatch, shape, gate_rows):
    """Which gates reach the kernels as they are, and that every broadcast gives torch's values and gradients."""
    from protein_clip_amd import ops
    g = torch.Generator().manual_seed(1)
    u = torch.randn(5, 12, 6, generator=g, dtype=torch.float32).requires_grad_(True)
    gate = torch.randn(shape, generator=g).requires_grad_(True)
    seen = []
    real = provider.norm_gate_fwd
    monkeypatch.setattr(provider, "norm_gate_fwd", lambda u, r, gt, rows, *a: seen.append((gt.numel(), rows)) or real(u, r, gt, rows, *a))
    y = ops.norm_gate_residual(u, gate=gate, after=(None, None), scale=2.0)
    want = R.normed(u, "layer", None, None, 1e-5) * gate * 2.0
    torch.testing.assert_close(y, want)
    assert seen == [(360 // gate_rows, gate_rows)] if gate_rows else seen == [(360, 1)]
    dy = torch.randn(5, 12, 6, generator=g)
    for a, b in zip(torch.autograd.grad(y, (u, gate), dy), torch.autograd.grad(want, (u, gate), dy)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


# ---- towers and loops --------------------------------------------------------------------------------------
HID, EMB = 24, 16


class _Trunk(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.table = torch.nn.Parameter(torch.randn(33, HID, generator=torch.Generator().manual_seed(11)), requires_grad=False)

    def forward(self, input_ids, attention_mask):
        return type("Out", (), {"last_hidden_state": self.table[input_ids]})()


def _model(kind, token_dtype=None, dropout=0.0):
    from protein_clip_amd.modules import models
    torch.manual_seed(0)
    return (models.ExtendedCLIP if kind == "clip" else models.ExtendedFILIP)(HID, EMB, 3, 2, dropout, _Trunk(), token_dtype)


def _batch():
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(4, 24, (4, 9), generator=g)
    mask = torch.ones(4, 9, dtype=torch.int64)
    mask[1, 5:] = 0
    return {"input_ids": ids, "attention_mask": mask}, {"input_ids": ids.flip(0), "attention_mask": mask.flip(0)}


@pytest.mark.parametrize("kind", ["clip", "filip"])
def test_towers_on_the_operators_equal_the_modules(provider, kind):
    """Same parameters, f32: outputs and every parameter's gradient of the fused token head against the PyTorch modules."""
    res = []
    for token_dtype in (None, torch.float32):
        model = _model(kind, token_dtype).train()
        a, b = model(*_batch())
        (a.square().sum() + (a * b).sum()).backward()
        res.append((a, b, {n: p.grad for n, p in model.named_parameters() if p.grad is not None}))
    torch.testing.assert_close(res[0][0], res[1][0])
    torch.testing.assert_close(res[0][1], res[1][1])
    assert set(res[0][2]) == set(res[1][2]) and len(res[0][2]) > 10
    for n in res[0][2]:
        torch.testing.assert_close(res[0][2][n], res[1][2][n], rtol=2e-4, atol=2e-5, msg=lambda m: f"{n}: {m}")


def test_tower_dropout_follows_the_generator(provider):
    model = _model("filip", torch.float32, dropout=0.5).train()
    outs = []
    for seed in (1, 1, 2):
        torch.manual_seed(seed)
        outs.append(model(*_batch())[0])
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])
    model.eval()
    assert torch.equal(model(*_batch())[0], model(*_batch())[0])
    with pytest.raises(ValueError, match="token_dtype"):
        _model("clip", torch.float64)


def _step(kind, pep, rec, limit, token_dtype=None):
    from protein_clip_amd import synthetic as S
    from protein_clip_amd.modules import training_utils, training_utils_filip
    mod = training_utils if kind == "clip" else training_utils_filip
    model = _model(kind, token_dtype)
    opt = torch.optim.SGD([p for p in model.parameters() if p.requires_grad], lr=1.0)
    before = {n: p.detach().clone() for n, p in model.named_parameters() if p.requires_grad}
    loss = mod.train(model, [(pep, rec)], opt, S.make_tokenizer(), "cpu", **({} if limit is None else {"max_grad_norm": limit}))
    return loss, {n: before[n] - p.detach() for n, p in model.named_parameters() if p.requires_grad}


def _pairs():
    from protein_clip_amd import synthetic as S
    return S.random_sequences(8, 4, 12, seed=5), S.random_sequences(8, 9, 30, seed=6)


def _norm(step):
    return torch.sqrt(sum((v.double() ** 2).sum() for v in step.values())).item()


@pytest.mark.parametrize("kind", ["clip", "filip"])
def test_loops_clip_the_gradient_norm(provider, kind):
    """One SGD step of rate one is the gradient: with a limit below its norm it is the same direction at the limit's length."""
    pep, rec = _pairs()
    loss, free = _step(kind, pep, rec, None)
    size = _norm(free)
    clipped_loss, clipped = _step(kind, pep, rec, 0.5 * size)
    assert clipped_loss == loss and abs(_norm(clipped) / (0.5 * size) - 1) < 1e-4
    for n in free:
        torch.testing.assert_close(clipped[n], 0.5 * free[n], rtol=1e-4, atol=1e-6 * size)
    _, loose = _step(kind, pep, rec, 10 * size)
    assert all(torch.equal(loose[n], free[n]) for n in free)


def test_big_batch_loop_clips_unscaled_gradients(provider):
    from torch.amp import GradScaler
    from protein_clip_amd import synthetic as S
    from protein_clip_amd.modules import training_utils
    pep, rec = _pairs()
    loader = [(pep[:4], rec[:4]), (pep[4:], rec[4:])]
    sizes = []
    for limit in (None, 0.01):
        model = _model("clip")
        opt = torch.optim.SGD([p for p in model.parameters() if p.requires_grad], lr=1.0)
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        training_utils.train_gc(model, loader, S.make_tokenizer(), opt, GradScaler("cpu", enabled=True, init_scale=1024.0), "cpu", 2, max_grad_norm=limit)
        sizes.append(_norm({n: before[n] - p.detach() for n, p in model.named_parameters()}))
    assert sizes[0] > 0.02 and abs(sizes[1] / 0.01 - 1) < 1e-3


def _worker(rank, port, out_dir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK=str(rank))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    import token_cpu_provider as P
    from protein_clip_amd import ops
    ops._hip_kernels = P
    pep, rec = _pairs()
    own = slice(rank * 4, rank * 4 + 4)
    torch.save({(k, d): _step(k, pep[own], rec[own], 0.05, getattr(torch, d) if d else None) for k in ("clip", "filip") for d in ("", "float32")},
               os.path.join(out_dir, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_clip_like_one_process(provider, tmp_path):
    """The gradients summed over two ranks are clipped by the norm of the sum: the step equals the single process's on the whole batch."""
    for attempt in range(3):
        with socket.socket() as sk:
            sk.bind(("127.0.0.1", 0))
            port = sk.getsockname()[1]
        try:
            mp.start_processes(_worker, args=(port, str(tmp_path)), nprocs=2, join=True, start_method="spawn")
            break
        except Exception as e:
            if attempt == 2 or not is_port_clash(e):
                raise
    pep, rec = _pairs()
    for rank in range(2):
        for (kind, d), (loss, step) in torch.load(tmp_path / f"rank{rank}.pt", weights_only=False).items():
            want_loss, want = _step(kind, pep, rec, 0.05, getattr(torch, d) if d else None)
            assert abs(loss - want_loss) < 2e-5 and abs(_norm(step) / 0.05 - 1) < 1e-3
            for n in want:
                torch.testing.assert_close(step[n], want[n], rtol=1e-3, atol=1e-6, msg=lambda m: f"{kind} {d} rank {rank} {n}: {m}")


def test_entry_options(monkeypatch):
    from protein_clip_amd import entry
    monkeypatch.setattr(sys, "argv", ["main.py"])
    args = entry.parse_args({"epochs": 1, "batch_size": 2})
    assert entry.TOKEN_DTYPES[args.token_dtype] is None and args.max_grad_norm is None
    monkeypatch.setattr(sys, "argv", ["main.py", "--token-dtype", "bf16", "--max-grad-norm", "1.5"])
    args = entry.parse_args({"epochs": 1, "batch_size": 2})
    assert entry.TOKEN_DTYPES[args.token_dtype] is torch.bfloat16 and args.max_grad_norm == 1.5


class _RawWriter:
    """Writes the tensors' memory as the kernels do: without torch knowing."""

    @staticmethod
    def grad_clip(src, dst=None, max_norm=0.0, eps=1e-6):
        norm = torch.sqrt(sum((t.detach().double() ** 2).sum() for t in src)).float()
        values = [t.detach() * torch.clamp(max_norm / (norm + eps), max=1.0) for t in src]
        for v, d in zip(values, dst):
            d.detach().numpy()[...] = v.numpy()
        return norm.reshape(1)


@pytest.mark.parametrize("where", ["in place", "out"])
def test_clipping_counts_as_a_write(where):
    """A backward that needs a value which clipping has overwritten is refused, as after torch's own in-place operations."""
    from protein_clip_amd import ops
    a = torch.ones(8, requires_grad=True)
    v = torch.ones(8)
    y = (a * v).sum()   # keeps v
    if where == "in place":
        ops.clip_grads([v], 0.5, kernels=_RawWriter)
    else:
        ops.clip_grads([torch.ones(8)], 0.5, out=[v], kernels=_RawWriter)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_clipping_tensors_of_inference_mode():
    """Tensors made in inference mode have no version; they are clipped with the others."""
    from protein_clip_amd import ops
    with torch.inference_mode():
        v = torch.ones(3)
    w = torch.ones(1)
    ops.clip_grads([v, w], 1.0, kernels=_RawWriter)
    assert abs(v[0].item() - 0.5) < 1e-6 and w._version == 1
