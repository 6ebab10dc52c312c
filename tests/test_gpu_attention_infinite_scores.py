"""Rows whose visible scores are all -inf: softmax of them is NaN, whether the row's keys are cut into splits or not. A part of
a row's scores at -inf only leaves those keys out."""
import math

import pytest
import torch

from sparseconv.ops.attention import sparse_attention

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def ends(*lengths):
    return torch.tensor([0, *lengths], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def inputs(n, m, H, D, dtype, hidden):
    """The scores of the keys of `hidden` are -inf for every query: -inf in a column where queries hold 1."""
    g = torch.Generator(device="cuda").manual_seed(n + m + D)
    q, k, v = (torch.randn(r, H, D, generator=g, device="cuda").to(dtype) for r in (n, m, m))
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[hidden, :, 0] = -math.inf
    return [t.requires_grad_() for t in (q, k, v)]


# one query over 20,000 keys is cut into splits, 3,000 queries of 64 heads are not
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m,H,D", [(1, 20000, 2, 64), (3, 20000, 1, 128), (3000, 200, 32, 64), (40, 70, 2, 33), (2, 9000, 2, 136)])
@pytest.mark.parametrize("causal", [False, True])
def test_all_scores_at_minus_infinity(dtype, n, m, H, D, causal):
    leaves = inputs(n, m, H, D, dtype, slice(None))
    out = sparse_attention(*leaves, ends(n), ends(m), causal=causal)
    seen = slice(max(0, n - m) if causal else 0, None)
    assert out[seen].isnan().all() and (out[:seen.start] == 0).all()
    gq, gk, gv = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert gv.isnan().all()
    if m > 1:
        assert gk.isnan().all() and gq[n - 1].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 3000])
def test_finite_inputs_whose_scores_overflow(dtype, n):
    """One query's products of 1e30 and -1e30 pass fp32's range; the others do not see that column."""
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k, v = (torch.randn(r, 2, 64, generator=g, device="cuda").to(dtype) for r in (n + 1, 20000, 20000))
    q[..., 0], k[..., 0] = 0.0, -1e30
    q[n, :, 0] = 1e30
    out = sparse_attention(q, k, v, ends(n + 1), ends(20000))
    assert out[n].isnan().all() and out[:n].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", [slice(0, 15000), slice(5000, None), slice(7, 19999)])
@pytest.mark.parametrize("D", [64, 128, 136])
def test_some_scores_at_minus_infinity(dtype, hidden, D):
    """Whole splits of them; the rest alone gives the same row."""
    q, k, v = (t.detach() for t in inputs(2, 20000, 2, D, dtype, hidden))
    out = sparse_attention(q, k, v, ends(2), ends(20000)).double()
    left = torch.ones(20000, dtype=torch.bool)
    left[hidden] = False
    s = torch.einsum("ihd,jhd->hij", q.double(), k[left].double()) * D ** -0.5
    want = torch.einsum("hij,jhd->ihd", s.softmax(-1), v[left].double())
    # p and the result rounded: half a step each; fp32: exponents to a few 2^-22
    assert (out - want).norm() < {torch.float32: 4e-6}.get(dtype, 2.0 * torch.finfo(dtype).eps) * want.norm()


@pytest.mark.parametrize("dtype", TYPES)
def test_samples_without_keys_beside_them(dtype):
    """In splits, rows that see no key stay zeros."""
    q, k, v = inputs(3, 20000, 2, 64, dtype, slice(None))
    out = sparse_attention(q, k, v, ends(1, 1, 1), ends(12000, 0, 8000))
    assert out[0].isnan().all() and (out[1] == 0).all() and out[2].isnan().all()
    gq, _, _ = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert (gq[1] == 0).all() and gq[0].isnan().all() and gq[2].isnan().all()
