"""Queries' gradients of narrow heads, where the roundings of ds add up along what a row's keys have in common: with ds in two parts
they are off by their own rounding and by what p's rounding in out leaves in grad . out, which is no more: as two independent errors,
sqrt(2) times the first at most."""
import math

import pytest
import torch

from sparseconv.ops.attention import sparse_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [8, 12, 16, 24, 32])
@pytest.mark.parametrize("n,m,H,K,causal", [(300, 257, 2, 2, False), (300, 64, 4, 1, False), (300, 300, 2, 1, True), (700, 1000, 2, 2, False)])
def test_queries_gradients(dtype, D, n, m, H, K, causal):
    samples = 12
    g = torch.Generator(device="cuda").manual_seed(m + D)
    q, k, v, grad = (torch.randn(samples, r, h, D, generator=g, device="cuda").mul_(s).to(dtype)
                     for r, h, s in ((n, H, 1.5), (m, K, 1.0), (m, K, 1.0), (n, H, 1.0)))
    ends = lambda rows: (torch.arange(samples + 1, device="cuda") * rows).int()
    leaves = [t.flatten(0, 1).requires_grad_() for t in (q, k, v)]
    out = sparse_attention(*leaves, ends(n), ends(m), causal=causal)
    (got,) = torch.autograd.grad(out, leaves[:1], grad.flatten(0, 1))
    a, d = (t.double().transpose(1, 2) for t in (q, grad))
    b, c = (t.double().repeat_interleave(H // K, 2).transpose(1, 2) for t in (k, v))
    s = a @ b.transpose(-1, -2) * D ** -0.5
    if causal:
        s = s.masked_fill(torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1), -math.inf)
    p, dp = s.softmax(-1), d @ c.transpose(-1, -2)
    want = ((p * (dp - (p * dp).sum(-1, keepdim=True))) @ b * D ** -0.5).transpose(1, 2).flatten(0, 1)
    own = (want.to(dtype).double() - want).norm()
    assert (got.double() - want).norm() < math.sqrt(2.0) * own, ((got.double() - want).norm() / own).item()
