"""CLIP train / eval loops and loss functions with the reference's names and signatures
(modules/training_utils.py).

``_contrastive_loss`` / ``_contrastive_loss_gc`` / ``get_logits`` run on the HIP kernels.
``train_gc`` keeps GradCache's semantics — no-grad forward of every sub-batch, ONE loss over
the concatenated representations, re-forward with the cached representation gradients — but
needs no ``grad_cache`` package, and when ``torch.distributed`` is initialised the
concatenation additionally spans every rank through an RCCL all-gather inside the loss
(each rank then back-propagates its own rows only; head gradients are summed over ranks).
"""
from __future__ import annotations

import torch
import torch.distributed as dist

from .. import ops


# --------------------------------------------------------------------------------------
# losses
# --------------------------------------------------------------------------------------
def _contrastive_loss(pep_embedding: torch.Tensor, rec_embedding: torch.Tensor) -> torch.Tensor:
    """Symmetric InfoNCE of ``pep_embedding [B,d] @ rec_embedding [d,B]``
    (training_utils.py:74-89; the caller passes ``rec.t()``)."""
    return ops.clip_loss(pep_embedding, rec_embedding.t())


def _cat(x):
    return torch.cat(list(x), dim=0) if isinstance(x, (list, tuple)) else x


def _contrastive_loss_gc(x, y, group=None) -> torch.Tensor:
    """Same loss on lists of sub-batch representations (training_utils.py:247-265); with a
    process group the batch is the concatenation over all ranks."""
    return ops.clip_loss(_cat(x), _cat(y), group=group)


def get_logits(x, y) -> torch.Tensor:
    """``exp(x @ y.T)`` of the concatenated lists (training_utils.py:157-172)."""
    return ops.clip_exp_logits(_cat(x), _cat(y))


# --------------------------------------------------------------------------------------
# plain loops
# --------------------------------------------------------------------------------------
def _tokenise(tokenizer, sequences, device):
    return tokenizer(sequences, return_tensors="pt", padding=True).to(device)


def _process_batch(model, batch_data, tokenizer, device, compute_grad=False, scaler=None):
    peptides, receptors = batch_data
    pep, rec = model(_tokenise(tokenizer, peptides, device), _tokenise(tokenizer, receptors, device))
    loss = _contrastive_loss(pep, rec.t())
    if compute_grad:
        _backward(loss, scaler)
    return loss.item()


def _loss_scaler(model, scaler, device):
    """The scaler that a loop's backward runs under: the caller's, or one of the loop's own where that scales nothing and the towers' token
    heads compute in float16: the gradients of a mean over batch and tokens, 1e-7 or so an element, would lie among float16's
    subnormal numbers (steps of 6e-8) or below them."""
    if scaler is not None and scaler.is_enabled():
        return scaler
    if any(getattr(m, "token_dtype", None) == torch.float16 for m in getattr(model, "modules", list)()):
        return torch.amp.GradScaler(torch.device(device).type)
    return scaler


def _backward(loss, scaler):
    (loss if scaler is None else scaler.scale(loss)).backward()


def _distributed() -> bool:
    return dist.is_available() and dist.is_initialized() and dist.get_world_size() > 1


def _clip(model, optimizer, max_grad_norm, scaler=None):
    """Clips the gradients of the model's parameters; under a scaler those that the optimizer steps, which are the ones it unscales."""
    parameters = model.parameters()
    if scaler is not None and scaler.is_enabled():
        scaler.unscale_(optimizer)
        parameters = [p for group in optimizer.param_groups for p in group["params"]]
    ops.clip_grad_norm_(parameters, max_grad_norm)


def _finish_step(model, optimizer, max_grad_norm=None, scaler=None):
    """What follows a backward: the sum over the ranks, when asked for the clipping of the global gradient norm (of the sum, so that
    every rank scales by the same factor, and without the loss's scale), and the optimizer's step."""
    scaled = scaler is not None and scaler.is_enabled()
    if _distributed():
        _sum_head_grads(model, max_grad_norm=None if scaled else max_grad_norm)
    if max_grad_norm is not None and (scaled or not _distributed()):
        _clip(model, optimizer, max_grad_norm, scaler)
    if scaled:
        scaler.step(optimizer)
        scaler.update()
    else:
        optimizer.step()


def train(model, data_loader, optimizer, tokenizer, device, max_grad_norm=None, scaler=None):
    """One epoch, one optimizer step per batch; returns the mean batch loss.  Under
    ``torch.distributed`` the loss of a batch spans the batches of all ranks (all-gather inside
    the loss) and every rank back-propagates its own rows, so the head gradients are summed over
    the ranks before the step.  ``max_grad_norm``: clip the global gradient norm to this (None: no clipping,
    as in the reference).  ``scaler``: a ``torch.amp.GradScaler`` for the loss; towers with float16 token heads get one for the
    epoch when there is none."""
    model.train()
    scaler = _loss_scaler(model, scaler, device)
    running = 0.0
    for batch in data_loader:
        optimizer.zero_grad()
        running += _process_batch(model, batch, tokenizer, device, compute_grad=True, scaler=scaler)
        _finish_step(model, optimizer, max_grad_norm, scaler)
    return running / len(data_loader)


def evaluate(model, data_loader, tokenizer, device):
    model.eval()
    running = 0.0
    with torch.no_grad():
        for batch in data_loader:
            running += _process_batch(model, batch, tokenizer, device)
    return running / len(data_loader)


# --------------------------------------------------------------------------------------
# big-batch training (GradCache semantics, optionally across ranks)
# --------------------------------------------------------------------------------------
class _RngSnapshot:
    """Random state of the CPU and of one GPU, so a sub-batch can be re-run with the very
    dropout masks of its first pass."""

    def __init__(self, device):
        self.cpu = torch.get_rng_state()
        self.dev = torch.device(device)
        self.cuda = torch.cuda.get_rng_state(self.dev) if self.dev.type == "cuda" else None

    def restore(self):
        torch.set_rng_state(self.cpu)
        if self.cuda is not None:
            torch.cuda.set_rng_state(self.cuda, self.dev)


def _encode_cached(encoder, inputs, device):
    """First pass of one sub-batch: representation without a graph (a leaf that will receive
    the loss gradient) plus what is needed to replay the pass."""
    snap = _RngSnapshot(device)
    with torch.no_grad():
        rep = encoder(inputs)
    return rep.detach().requires_grad_(True), snap


def _replay(encoder, inputs, snap, rep):
    """Second pass with a graph under the first pass's random state; pushes the cached
    representation gradient through it (the surrogate is <rep_again, d loss / d rep>)."""
    keep = _RngSnapshot(snap.dev)
    snap.restore()
    again = encoder(inputs)
    keep.restore()
    torch.autograd.backward(again, grad_tensors=rep.grad)


def _sum_head_grads(model, group=None, max_grad_norm=None):
    """Every rank back-propagated the global loss through its own rows only, so the gradient
    of a shared parameter is the SUM over ranks (one flat all-reduce).  With ``max_grad_norm`` the way back from the
    flat buffer clips as well."""
    grads = [p.grad for p in model.parameters() if p.requires_grad and p.grad is not None]
    if not grads:
        return
    flat = torch.cat([g.reshape(-1) for g in grads])
    dist.all_reduce(flat, group=group)
    parts = [v.view(g.shape) for v, g in zip(flat.split([g.numel() for g in grads]), grads)]
    if max_grad_norm is not None:
        # straight into the gradients; one of another layout than its part is clipped in the part and copied like the others without clipping
        ops.clip_grads(parts, max_grad_norm, out=[g if g.is_contiguous() else v for v, g in zip(parts, grads)])
    for v, g in zip(parts, grads):
        if max_grad_norm is None or not g.is_contiguous():
            g.copy_(v)


def train_gc(model, data_loader, tokenizer, optimizer, scaler, device, accumulated_batches=1, group=None, max_grad_norm=None):
    """Big-batch epoch (training_utils.py:92-155): every ``accumulated_batches`` sub-batches
    form one contrastive batch and one optimizer step.  Trailing sub-batches that do not fill
    a batch are encoded and dropped, as in the reference.  ``max_grad_norm``: as in :func:`train`, applied to
    the unscaled gradients.  ``scaler``: one that is not enabled is replaced, for the epoch, where the towers' token heads are
    float16.  Returns the mean big-batch loss."""
    model.train()
    scaler = _loss_scaler(model, scaler, device)
    distributed = _distributed()
    total, big_batches = 0.0, 0
    pending = []
    for step, (xx, yy) in enumerate(data_loader):
        xx = _tokenise(tokenizer, xx, device)
        yy = _tokenise(tokenizer, yy, device)
        xx["temperature"] = model.temperature
        yy["temperature"] = model.temperature
        rx, sx = _encode_cached(model.pep_encoder, xx, device)
        ry, sy = _encode_cached(model.rec_encoder, yy, device)
        pending.append((xx, yy, rx, ry, sx, sy))
        if (step + 1) % accumulated_batches:
            continue
        big_batches += 1
        print(step)
        loss = _contrastive_loss_gc([p[2] for p in pending], [p[3] for p in pending], group=group if distributed else None)
        total += loss.item()
        scaler.scale(loss).backward()
        for xx_, yy_, rx_, ry_, sx_, sy_ in pending:
            _replay(model.pep_encoder, xx_, sx_, rx_)
            _replay(model.rec_encoder, yy_, sy_, ry_)
        pending = []
        if distributed:
            _sum_head_grads(model, group)
        if max_grad_norm is not None:
            _clip(model, optimizer, max_grad_norm, scaler)
        scaler.step(optimizer)
        scaler.update()
        optimizer.zero_grad()
    return total / max(big_batches, 1)


def eval_gc_allrec_onepep(model, data_loader, device, tokenizer, agg_batches=2, k=0):
    """Rank of peptide ``k`` against the receptors of the first ``agg_batches`` sub-batches
    (training_utils.py:174-228): every row of the score matrix is that one peptide, so the
    diagonal holds its score against each receptor; returns ``[1 + number of receptors scoring
    higher than receptor k]`` after the first aggregated batch, like the reference."""
    model.eval()
    chosen, seen = None, 0
    for xx, yy in data_loader:
        if k // len(xx) == seen:
            chosen = xx[k % len(yy)]
        seen += 1
    reps_x, reps_y, ranks = [], [], []
    with torch.no_grad():
        for step, (xx, yy) in enumerate(data_loader):
            xx = _tokenise(tokenizer, (chosen,) * len(xx), device)
            yy = _tokenise(tokenizer, yy, device)
            xx["temperature"] = model.temperature
            yy["temperature"] = model.temperature
            reps_x.append(model.pep_encoder(xx))
            reps_y.append(model.rec_encoder(yy))
            if (step + 1) % agg_batches == 0:
                scores = torch.diag(get_logits(reps_x, reps_y))
                ranks.append(int((scores > scores[k]).sum().item()) + 1)
                return ranks
    return ranks
