"""GPU tests of the paths that call the token-head operators: the towers with ``token_dtype`` and the loops with ``max_grad_norm``."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import protein_clip_amd  # noqa: F401
    from protein_clip_amd import synthetic
    return synthetic


def _model(S, kind, token_dtype, dropout=0.0):
    from protein_clip_amd.modules import models
    torch.manual_seed(0)
    esm = S.make_esm(64, 1, 4)
    for p in esm.parameters():
        p.requires_grad = False
    return (models.ExtendedCLIP if kind == "clip" else models.ExtendedFILIP)(64, 32, 3, 2, dropout, esm, token_dtype).cuda()


def _batch(S):
    tok = S.make_tokenizer()
    make = lambda lo, hi, seed: tok(S.random_sequences(6, lo, hi, seed), return_tensors="pt", padding=True).to("cuda")
    return make(4, 12, 1), make(9, 40, 2)


@pytest.mark.parametrize("kind", ["clip", "filip"])
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 0.08), (torch.float16, 0.01)])
def test_token_head_against_the_modules(S, kind, dtype, tol):
    """Per-residue embeddings and the parameter gradients of the fused token head against the PyTorch modules in 32 bits.  Five results
    forward and five backward carry a rounding (half a step) of their own and of their operand's: 2 * 10 half steps of the type,
    0.08 for bfloat16, 0.01 for float16; float32 differs by the order of its sums only.

    Gradients pass two ReLUs as well, whose slope is the other one where an error moved the input across zero: inputs spread like
    a normal variable and off by four half steps h lie so near to zero with probability 2 * 0.4 * 4 h, and a sum of which that
    share of the terms is dropped or added is off by the root of the share: sqrt(3.2 h) for each ReLU (h = 2^-8: 0.11, 2^-11: 0.04)."""
    from protein_clip_amd.modules import models
    res = []
    for d in (None, dtype):
        model = _model(S, kind, d).eval()
        tower, seq = model.rec_encoder, _batch(S)[1]
        h = models._token_features(tower, seq)
        assert h.dtype == torch.float32
        weight = torch.cos(torch.arange(h.numel(), device="cuda")).view(h.shape)
        names, params = zip(*[(n, p) for n, p in tower.named_parameters() if "projection" in n or "amino_acid" in n])
        res.append((h, dict(zip(names, torch.autograd.grad((h * weight).sum(), params)))))
    off = lambda a, b: ((a - b).double().norm() / b.double().norm()).item()
    assert off(res[1][0], res[0][0]) <= tol
    crossed = 0.0 if dtype == torch.float32 else 2 * (3.2 * torch.finfo(dtype).eps / 2) ** 0.5
    for n, g in res[0][1].items():
        assert res[1][1][n].dtype == torch.float32 and off(res[1][1][n], g) <= tol + crossed, n


@pytest.mark.parametrize("kind", ["clip", "filip"])
def test_training_with_token_dtype_and_clipping(S, kind):
    """The loops run on the operators; the step taken (SGD of rate one) has the limit's length, or the gradient's own."""
    from protein_clip_amd.modules import training_utils, training_utils_filip
    mod = training_utils if kind == "clip" else training_utils_filip
    pairs = [(S.random_sequences(6, 4, 12, 1), S.random_sequences(6, 9, 40, 2))]
    for limit in (None, 1e-3):
        model = _model(S, kind, torch.bfloat16, dropout=0.1)
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        opt = torch.optim.SGD([p for p in model.parameters() if p.requires_grad], lr=1.0)
        loss = mod.train(model, pairs, opt, S.make_tokenizer(), "cuda", max_grad_norm=limit)
        assert loss == loss
        size = torch.sqrt(sum(((before[n] - p).double() ** 2).sum() for n, p in model.named_parameters())).item()
        # a step of 1e-3 subtracted from parameters of order 0.1 in 32 bits: each is off by 2^-24 * 0.2 at most, 10,000 of them by 1.2e-6 together
        assert size > 2e-3 if limit is None else abs(size / limit - 1) < 5e-3
