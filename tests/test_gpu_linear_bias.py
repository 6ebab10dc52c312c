"""An fp32 bias of a 16-bit layer is added as it is: with products of zero and the negative of the rounded bias
as residual, the output is what the rounding would have lost (exact in fp32), rounded once."""
import pytest
import torch

from sparseconv import _native
from sparseconv.ops.linear import sparse_linear

pytestmark = pytest.mark.gpu


# on tensor cores with W resident, streamed, over pairs of CTAs and with more columns than shared memory keeps; on the
# CUDA cores; through copies into whole rows
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,Ci,Co", [(1, 8, 8), (300, 64, 72), (50000, 64, 256), (3000, 1024, 256), (20000, 512, 520), (200, 64, 5000),
                                     (100, 35, 13), (5, 16, 5), (20000, 257, 131), (60000, 72, 93)])
def test_added_unrounded(M, Ci, Co, dtype):
    g = torch.Generator(device="cuda").manual_seed(Co)
    x = torch.randn(M, Ci, generator=g, device="cuda").to(dtype)
    w = torch.zeros(Co, Ci, device="cuda")
    for b in (torch.rand(Co, generator=g, device="cuda") + 0.5, (torch.rand(Co, generator=g, device="cuda").double() + 0.5)):
        r = -b.to(dtype).expand(M, Co).contiguous()
        want = (b.float() + r[0].float()).to(dtype).expand(M, Co)
        assert (want != 0).float().mean() > 0.7
        for act in ("none", "relu"):
            assert torch.equal(sparse_linear(x, w, b, residual=r, activation=act), want)
    leaf = b.float().requires_grad_(True)
    out = sparse_linear(x, w, leaf, residual=r)
    assert torch.equal(out.detach(), want)
    grad = torch.autograd.grad(out, leaf, torch.ones_like(out))[0]
    assert grad.dtype == torch.float32 and (grad == M).all()


def test_bias_types():
    x, w = torch.randn(4, 16, device="cuda", dtype=torch.float16), torch.randn(8, 16, device="cuda", dtype=torch.float16)
    b = torch.randn(8, device="cuda", dtype=torch.bfloat16)
    want = (x.float() @ w.float().t() + b.float())
    assert torch.allclose(sparse_linear(x, w, b).float(), want, rtol=2e-3, atol=2e-3)     # to fp32, exactly
    with pytest.raises(TypeError, match="bias"):
        _native.linear_forward(x, w, b, None, "none")
    with pytest.raises(TypeError, match="bias"):
        _native.linear_forward(x.float(), w.float(), b, None, "none")
