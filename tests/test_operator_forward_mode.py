"""Forward-mode derivatives through the linear, norm and clipping calls: they have none, and say so
rather than hand back a result without a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from sparseconv.ops.clip import clip_grad_norm_, clip_gradients
from sparseconv.ops.linear import sparse_linear
from sparseconv.ops.norm import sparse_norm, sparse_residual_norm

X, W, B = torch.randn(4, 8), torch.randn(8, 8), torch.randn(8)


def _param(grad):
    p = torch.nn.Parameter(torch.zeros(4, 8))
    p.grad = grad
    return p


CALLS = {
    "feats": lambda d: sparse_linear(d(X), W), "weight": lambda d: sparse_linear(X, d(W)),
    "bias": lambda d: sparse_linear(X, W, d(B)), "residual": lambda d: sparse_linear(X, W, residual=d(X)),
    "norm": lambda d: sparse_norm(d(X)), "norm_weight": lambda d: sparse_norm(X, d(B)),
    "step": lambda d: sparse_residual_norm(X, d(X)), "gate": lambda d: sparse_residual_norm(X, X, gate=d(B)),
    "next": lambda d: sparse_residual_norm(X, next_bias=d(B)),
    "clip": lambda d: clip_gradients([X.clone(), d(X)], 1.0), "out": lambda d: clip_gradients([X], 1.0, out=[d(X.clone())]),
    "clip_parameter": lambda d: clip_grad_norm_([_param(d(X))], 1.0),
}


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(name, grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match="no CPU fallback"):       # no tangent: as outside of the level
            CALLS[name](lambda t: t)


@pytest.mark.parametrize("f", [lambda x: sparse_linear(x, W), sparse_norm])
def test_jvp_is_refused(f):
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (X,), (torch.ones_like(X),))
