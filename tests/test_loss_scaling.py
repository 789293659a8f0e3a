"""CPU tests of the loops with float16 token heads, whose gradients need a scaled loss: on the test-only provider, with a temperature that
makes the gradients as small as those of a mean over a large batch."""
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

import test_token_ops_host as H  # noqa: E402


@pytest.fixture()
def provider():
    import token_cpu_provider as P
    from protein_clip_amd import ops
    real = ops._hip_kernels
    ops._hip_kernels = P
    yield P
    ops._hip_kernels = real


class _Recorder(torch.optim.SGD):
    """Keeps the gradients that each step is taken with."""

    def __init__(self, params):
        super().__init__(params, lr=0.0)
        self.seen = []

    def step(self, closure=None):
        self.seen.append({p: p.grad.clone() for p in self.param_groups[0]["params"] if p.grad is not None})
        return super().step(closure)


def _small(kind, token_dtype):
    """A model whose loss has a gradient of 5e-8 to 2e-6 an element of the per-residue embeddings, as a mean over some hundred pairs of some
    hundred tokens does: the scores are scaled by exp(t), or divided by t."""
    model = H._model(kind, token_dtype)
    with torch.no_grad():
        model.temperature.fill_(-8.0 if kind == "clip" else 2.0e3)
    return model


def _heads(model, grads=None):
    return {n: (p.grad if grads is None else grads[p]) for n, p in model.named_parameters() if "projection" in n or "amino_acid" in n}


def _grads(kind, token_dtype, pep, rec, limit=None, scaler=None, big_batch=False):
    """The gradients that one step of the loops is taken with, of the token heads' parameters."""
    from protein_clip_amd import synthetic as S
    from protein_clip_amd.modules import training_utils, training_utils_filip
    mod = training_utils if kind == "clip" else training_utils_filip
    model = _small(kind, token_dtype)
    opt = _Recorder([p for p in model.parameters() if p.requires_grad])
    if big_batch:
        half = len(pep) // 2
        mod.train_gc(model, [(pep[:half], rec[:half]), (pep[half:], rec[half:])], S.make_tokenizer(), opt, scaler, "cpu", 2, max_grad_norm=limit)
    else:
        mod.train(model, [(pep, rec)], opt, S.make_tokenizer(), "cpu", max_grad_norm=limit, **({} if scaler is None else {"scaler": scaler}))
    assert len(opt.seen) == 1, "the step was skipped"
    return _heads(model, opt.seen[0])


def _by_hand(kind, pep, rec):
    """The same float16 model's gradients with a loss scaled by 2^20."""
    from protein_clip_amd import synthetic as S
    from protein_clip_amd.modules import training_utils, training_utils_filip
    mod = training_utils if kind == "clip" else training_utils_filip
    model, tok = _small(kind, torch.float16), S.make_tokenizer()
    a, b = model(tok(pep, return_tensors="pt", padding=True), tok(rec, return_tensors="pt", padding=True))
    loss = mod._contrastive_loss(a, b.t()) if kind == "clip" else mod._compute_loss(a, b)
    (loss * 2.0 ** 20).backward()
    return {n: g / 2.0 ** 20 for n, g in _heads(model).items()}


def _off(a, b):
    """Relative distance of all gradients together."""
    num = sum(((a[n].double() - b[n].double()) ** 2).sum() for n in b)
    return (num / sum((b[n].double() ** 2).sum() for n in b)).sqrt().item()


# scaled by powers of two, the same bits go through both backward passes but for what is still subnormal: a hundredth at most, as for the
# roundings of all ten results in test_gpu_token_towers.py
TOL = 0.01
# against the modules in 32 bits a ReLU's slope is the other one for a share of the units (see there)
CROSSED = TOL + 2 * (3.2 * torch.finfo(torch.float16).eps / 2) ** 0.5


@pytest.mark.parametrize("kind", ["clip", "filip"])
def test_small_gradients_of_float16_heads_survive(provider, kind):
    pep, rec = H._pairs()
    want = _by_hand(kind, pep, rec)
    if kind == "clip":   # (FILIP's best partners of a token change with a rounding)
        assert _off(want, _grads(kind, None, pep, rec)) < CROSSED
    for scaler in (None, torch.amp.GradScaler("cpu", enabled=False), torch.amp.GradScaler("cpu", init_scale=2.0 ** 18)):
        assert _off(_grads(kind, torch.float16, pep, rec, scaler=scaler), want) < TOL


@pytest.mark.parametrize("kind", ["clip", "filip"])
def test_clipping_follows_the_unscaling(provider, kind):
    """The limit is compared with the norm of the gradients, not of the scaled ones: a quarter of it leaves a quarter."""
    pep, rec = H._pairs()
    free = _grads(kind, torch.float16, pep, rec)
    size = torch.sqrt(sum((g.double() ** 2).sum() for g in free.values())).item()
    loose, tight = (_grads(kind, torch.float16, pep, rec, limit=v) for v in (1e3, 0.0))
    assert _off(loose, free) < 1e-6 and not any(g.any() for g in tight.values())
    limited = _grads(kind, torch.float16, pep, rec, limit=size)   # the norm of all parameters is at least that of the heads'
    factor = limited[next(iter(free))].norm() / free[next(iter(free))].norm()
    assert 0 < factor <= 1 and _off(limited, {n: g * factor for n, g in free.items()}) < 1e-5


def test_small_gradients_in_the_big_batch_loop(provider):
    pep, rec = H._pairs()
    want = _by_hand("clip", pep, rec)
    for scaler in (torch.amp.GradScaler("cpu", enabled=False), torch.amp.GradScaler("cpu", init_scale=2.0 ** 18)):
        assert _off(_grads("clip", torch.float16, pep, rec, scaler=scaler, big_batch=True), want) < TOL


def test_other_types_are_not_scaled(provider):
    """Loops of float32 and bfloat16 towers run as before: no scaler of the loop's own, and a disabled one does nothing."""
    from protein_clip_amd.modules import training_utils as U
    for d in (None, torch.float32, torch.bfloat16):
        assert U._loss_scaler(H._model("clip", d), None, "cpu") is None
        off = torch.amp.GradScaler("cpu", enabled=False)
        assert U._loss_scaler(H._model("clip", d), off, "cpu") is off
    on = torch.amp.GradScaler("cpu")
    assert U._loss_scaler(H._model("clip", torch.float16), on, "cpu") is on


def _worker(rank, port, out_dir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK=str(rank))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    import token_cpu_provider as P
    from protein_clip_amd import ops
    ops._hip_kernels = P
    pep, rec = H._pairs()
    own = slice(rank * 4, rank * 4 + 4)
    torch.save({k: _grads(k, torch.float16, pep[own], rec[own]) for k in ("clip", "filip")}, os.path.join(out_dir, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_scale_like_one_process(provider, tmp_path):
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
    pep, rec = H._pairs()
    ranks = [torch.load(tmp_path / f"rank{r}.pt", weights_only=True) for r in range(2)]
    for kind in ("clip", "filip"):
        assert all(torch.equal(ranks[0][kind][n], ranks[1][kind][n]) for n in ranks[0][kind])
        assert _off(ranks[0][kind], _by_hand(kind, pep, rec)) < TOL
