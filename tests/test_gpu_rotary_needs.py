"""Queries and keys of which one needs a gradient: the other's turned values are constants, as it is."""
import pytest
import torch

from sparseconv.ops.attention import sparse_attention
from sparseconv.ops.rotary import sparse_rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 1])
def test_one_of_two_needs_a_gradient(which):
    pair = [torch.randn(50, 2, 32, device="cuda") for _ in range(2)]
    v, pos = torch.randn(50, 2, 32, device="cuda"), torch.arange(50, device="cuda", dtype=torch.int32)
    pair[which].requires_grad_()
    turned = sparse_rotary(*pair, pos)
    assert turned[which].requires_grad and not turned[1 - which].requires_grad
    grad = torch.randn(50, 2, 32, device="cuda")
    (got,) = torch.autograd.grad(sparse_attention(*turned, v), pair[which], grad)
    both = [t.detach().clone().requires_grad_() for t in pair]
    want = torch.autograd.grad(sparse_attention(*sparse_rotary(*both, pos), v), both, grad)[which]
    assert torch.equal(got, want)


def test_both_need_one():
    pair = [torch.randn(50, 2, 32, device="cuda", requires_grad=True) for _ in range(2)]
    pos = torch.arange(50, device="cuda", dtype=torch.int32)
    q, k = sparse_rotary(*pair, pos)
    assert q.requires_grad and k.requires_grad
    (got,) = torch.autograd.grad(q, pair[0], torch.ones_like(q))
    (alone,) = torch.autograd.grad(sparse_rotary(pair[0], None, pos)[0], pair[0], torch.ones_like(q))
    assert torch.equal(got, alone)
