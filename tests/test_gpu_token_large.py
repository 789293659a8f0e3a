"""GPU tests of the token-head operators on operands of more than 2^31 elements (offsets beyond 32 bits): the last rows, and sums that
reach them, against the same rows alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import protein_clip_amd  # noqa: F401
    from protein_clip_amd import ops as _ops
    yield _ops
    torch.cuda.empty_cache()


def test_linear_beyond_32_bit_offsets(ops):
    """4.4 GB of input rows, then 4.4 GB of output rows; everything but the last rows is zero."""
    for rows, width, out in ((2**31 // 640 + 100, 640, 16), (2**31 // 640 + 100, 16, 640)):
        x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
        x[-70:] = torch.randn(70, width, generator=torch.Generator().manual_seed(0)).to(x)
        w = (torch.randn(out, width, generator=torch.Generator().manual_seed(1)) * 0.1).to(x)
        y = ops.linear_act(x, w, activation="none")
        assert torch.equal(y[-70:], ops.linear_act(x[-70:].clone(), w)) and not y[:70].any()
        del y
        leaf = w.clone().requires_grad_(True)
        small = w.clone().requires_grad_(True)
        a = ops.linear_act(x, leaf)
        g, = torch.autograd.grad(a, leaf, torch.ones_like(a))
        del a
        b = ops.linear_act(x[-70:].clone(), small)
        h, = torch.autograd.grad(b, small, torch.ones_like(b))
        # the same 70 products in another order, rounded once: a step of bfloat16
        torch.testing.assert_close(g, h, rtol=2.0 ** -7, atol=1e-3)
        del x, g


def test_norm_gate_beyond_32_bit_offsets(ops):
    rows, d = 2**31 // 640 + 50, 640
    u = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    u[-50:] = torch.randn(50, d, generator=torch.Generator().manual_seed(0)).to(u)
    w = torch.ones(d, device="cuda", requires_grad=True)
    y = ops.norm_gate_residual(u, after=(w, None))
    alone = ops.norm_gate_residual(u[-50:].clone(), after=(w, None))
    assert torch.equal(y[-50:], alone) and not y[:50].any()
    g, = torch.autograd.grad(y, w, torch.ones_like(y))
    h, = torch.autograd.grad(alone, w, torch.ones_like(alone))
    torch.testing.assert_close(g, h, rtol=1e-4, atol=1e-4)


def test_clip_beyond_32_bit_offsets(ops):
    big = torch.zeros(2**31 + 10_000, dtype=torch.bfloat16, device="cuda")
    big[-3:] = torch.tensor([3.0, 4.0, 12.0], dtype=torch.bfloat16)
    big[0] = 84.0
    assert ops.clip_grads([big], 8.5).item() == 85.0
    torch.testing.assert_close(big[[0, -3, -2, -1]].float(), torch.tensor([8.4, 0.3, 0.4, 1.2], device="cuda"), rtol=2.0 ** -8, atol=0)
