"""GPU tests of the ways in which the token-head operators are called: traced, in forward mode, from loops with float16 towers, with operands at
the far end of what they accept."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import protein_clip_amd  # noqa: F401
    from protein_clip_amd import ops as _ops
    return _ops


@pytest.mark.filterwarnings("ignore")
def test_traced_and_in_forward_mode(ops):
    """A trace gives the operators' results on new inputs; a tangent is refused."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(0)
    w, one = torch.randn(24, 40, generator=g).cuda(), torch.ones(40, device="cuda")
    calls = (lambda x: ops.linear_act(x, w, activation="silu"), lambda x: ops.norm_gate_residual(x, x, after=(one, None), before=(None, None))[1])
    for call in calls:
        traced = torch.jit.trace(call, (torch.randn(5, 40, generator=g).cuda(),))
        x = torch.randn(5, 40, generator=g).cuda()
        assert torch.equal(traced(x), call(x))
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, x))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        ops.grad_norm([forward_ad.make_dual(x, x)])
