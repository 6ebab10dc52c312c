"""Causal rows and the infinities and NaN of keys that they do not see: sums go over the keys that a row sees, and so do the
gradients' over the rows that see a key."""
import math

import pytest
import torch

from sparseconv import _native
from sparseconv.ops.attention import sparse_attention

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
#: queries, keys, heads, key heads: one tile, several, shared keys, splits, long enough for two tiles a block at D = 128
SHAPES = [(100, 100, 2, 2), (300, 300, 4, 2), (64, 3000, 2, 1), (200, 150, 2, 2), (1500, 1500, 20, 10), (9, 4, 8, 1)]


def tolerance(dtype):
    """Four roundings of half a step each; fp32: exponents to a few 2^-22, sums of some thousand terms."""
    return {torch.float32: 4e-6}.get(dtype, 2.0 * torch.finfo(dtype).eps)


def reference(q, k, v, grad):
    """In 64 bits, of finite inputs."""
    n, m, G = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    b, c = (t.repeat_interleave(G, 1) for t in leaves[1:])
    hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
    s = torch.einsum("ihd,jhd->hij", leaves[0], b) * q.shape[2] ** -0.5
    p = s.masked_fill(hidden, -math.inf).softmax(-1).masked_fill(hidden.all(1)[:, None], 0.0)
    out = torch.einsum("hij,jhd->ihd", p, c)
    return [out.detach(), *torch.autograd.grad(out, leaves, grad.double())]


def near(got, want, dtype):
    assert got.isfinite().all()
    norm = want.norm().item()
    assert (got.double() - want).norm().item() <= tolerance(dtype) * norm if norm else (got == 0).all()


def setup(n, m, H, K, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + m + D)
    return [torch.randn(r, h, D, generator=g, device="cuda").to(dtype) for r, h in ((n, H), (m, K), (m, K), (n, H))]


def run(q, k, v, grad, kernel=None):
    if kernel is not None:
        out, stats, args = _native.attention_forward(q, k, v, None, None, True, q.shape[2] ** -0.5, keep_stats=True, kernel=kernel)
        return [out, *_native.attention_backward_of(args, q, k, v, None, None, out, stats, grad, (True,) * 3)]
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = sparse_attention(*leaves, causal=True)
    return [out.detach(), *torch.autograd.grad(out, leaves, grad)]


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128, 136])
@pytest.mark.parametrize("shape", SHAPES)
def test_keys_that_rows_do_not_see(shape, D, dtype, value):
    n, m, H, K = shape
    q, k, v, grad = setup(n, m, H, K, D, dtype)
    want = reference(q, k, v, grad)
    first = m - min(n, m) + min(n, m) // 2 + 1                 # the first key that is not as it should be: hidden from half of the rows
    clean = first - m + n                                    # the rows before this one do not see it
    bad = v.clone()
    bad[first:, :, D // 2] = value
    out, gq, _, _ = run(q, k, bad, grad)
    near(out[:clean], want[0][:clean], dtype)
    near(gq[:clean], want[1][:clean], dtype)
    others = torch.arange(D, device="cuda") != D // 2
    near(out[clean:][..., others], want[0][clean:][..., others], dtype)
    if clean < n:
        column = out[clean:, :, D // 2]
        assert (column.isnan() if math.isnan(value) else ~column.isfinite()).all()
    bad = k.clone()
    bad[first:, :, D // 2] = value
    out, gq, _, _ = run(q, bad, v, grad)
    near(out[:clean], want[0][:clean], dtype)
    near(gq[:clean], want[1][:clean], dtype)
    assert not gq[clean:].isfinite().all(-1).any()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128, 136])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_that_do_not_see_a_key(shape, D, dtype, value):
    n, m, H, K = shape
    q, k, v, grad = setup(n, m, H, K, D, dtype)
    rows = max(0, n - m) + min(n, m) // 2                      # as many queries first that are not as they should be
    clean = rows + m - n                                     # the first key that none of them sees
    good = grad.clone()
    good[:rows] = 0.0
    want = reference(q, k, v, good)
    bad = grad.clone()
    bad[:rows, :, D // 2] = value
    _, gq, gk, gv = run(q, k, v, bad)
    near(gq[rows:], want[1][rows:], dtype)
    near(gk[clean:], want[2][clean:], dtype)
    near(gv[clean:], want[3][clean:], dtype)
    if clean > 0:
        assert not gv[:clean, :, D // 2].isfinite().any()
    bad = q.clone()
    bad[:rows, :, D // 2] = value
    out, gq, gk, gv = run(bad, k, v, grad)
    near(out[rows:], want[0][rows:], dtype)
    near(gq[rows:], want[1][rows:], dtype)
    near(gk[clean:], want[2][clean:], dtype)
    near(gv[clean:], want[3][clean:], dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_before_the_first_key(dtype):
    """They see nothing, and whatever their gradients hold goes nowhere."""
    q, k, v, grad = setup(200, 120, 2, 2, 64, dtype)
    want = reference(q, k, v, grad)
    bad, bad_q = grad.clone(), q.clone()
    bad[:80], bad_q[:80] = math.nan, math.inf
    got = run(bad_q, k, v, bad)
    assert (got[0][:80] == 0).all() and (got[1][:80] == 0).all()
    for a, b in zip(got, want):
        near(a, b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128, 136])
def test_a_row_that_sees_one_key_and_is_lost(dtype, D):
    """Its score has no gradient, so its query has none but of what it sees."""
    q, k, v, grad = setup(200, 200, 2, 2, D, dtype)
    q[0], k[1:] = math.nan, math.nan
    _, gq, _, _ = run(q, k, v, grad)
    assert (gq[0] == 0).all() and gq[1:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D", [(700, 64), (700, 128), (130, 136)])
def test_all_values_lost(dtype, n, D):
    """NaN everywhere, as after a step that overflowed: every row that sees one is NaN."""
    q, k, v, grad = setup(n, n, 2, 2, D, dtype)
    out, gq, gk, gv = run(q, k, torch.full_like(v, math.nan), grad)
    assert out.isnan().all() and gq[1:].isnan().all() and gk.isnan().all()
    out, gq, gk, gv = run(q, k, v, torch.full_like(grad, math.nan))
    assert gv.isnan().all() and gq[1:].isnan().all() and gk.isnan().all()
