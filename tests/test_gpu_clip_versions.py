"""Clipping writes its outputs where torch cannot see it: the tensors' versions have to count it, so that
a backward that still needs the old values raises instead of using the new ones."""
import pytest
import torch

from sparseconv.ops.clip import clip_grad_norm_, clip_gradients

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_norm", [0.1, 1e9])
def test_outputs_count_as_changed(max_norm):
    """In place or not, and whether or not the factor is one."""
    mine, grads = ([torch.randn(n, device="cuda", dtype=t) for n, t in ((100, torch.float32), (7, torch.float16))]
                   for _ in range(2))
    outs = [torch.empty_like(g) for g in grads]
    before = [[t._version for t in ts] for ts in (mine, grads, outs)]
    clip_gradients(mine, max_norm)
    clip_gradients(grads, max_norm, out=outs)
    for ts, old, changed in zip((mine, grads, outs), before, (True, False, True)):
        assert all((t._version > v) == changed for t, v in zip(ts, old))


def test_backward_that_needs_the_old_gradients_raises():
    x = torch.randn(50, device="cuda", requires_grad=True)
    (x ** 3).sum().backward(create_graph=True)
    penalty = x.grad.square().sum()                    # keeps x.grad for its backward
    clip_grad_norm_([x], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(penalty, x)


def test_inference_tensors():
    with torch.inference_mode():
        g = torch.randn(100, device="cuda")
        keep = g.clone()
        total = clip_gradients([g], 0.1)
        assert torch.allclose(g, keep * (0.1 / total), rtol=1e-5)
