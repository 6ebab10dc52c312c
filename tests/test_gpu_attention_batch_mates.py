"""What a sample's gradients may not depend on: the other samples of its batch."""
import math

import pytest
import torch

from sparseconv.ops.attention import sparse_attention

pytestmark = pytest.mark.gpu


def ends(lengths):
    return torch.tensor([0, *lengths], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def gradients64(q, k, v, grad, causal=False, rows=None):
    """Of one sample, in 64 bits; of the first `rows` queries alone for the queries'."""
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    s = torch.einsum("ihd,jhd->hij", leaves[0], leaves[1]) * q.shape[2] ** -0.5
    if causal:
        s = s.masked_fill(torch.ones(q.shape[0], k.shape[0], dtype=torch.bool, device=q.device).triu(1), -math.inf)
    out = torch.einsum("hij,jhd->ihd", s.softmax(-1), leaves[2])
    return torch.autograd.grad(out, leaves, grad.double())


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def small_step(want):
    """Half of fp16's smallest step over a result's root mean square: what rounding to fp16 takes from small results."""
    return 2.0 ** -25 / (want.norm().item() / want.numel() ** 0.5)


@pytest.mark.parametrize("mate", ["nan", "inf", "large", "no keys", "no queries"])
@pytest.mark.parametrize("D", [64, 128, 33])
@pytest.mark.parametrize("first", [False, True])
def test_small_fp16_gradients_beside_others(mate, D, first):
    """3,000 rows with gradients of 2^-12: ds of about 2^-24 needs its lift whatever else is in the batch. `unseen`: queries in
    the sample itself that see no key. Bound: two roundings, and the results' own smallest step."""
    n, other, H = 3000, 200, 2
    g = torch.Generator(device="cuda").manual_seed(D)
    make = lambda r: torch.randn(r, H, D, generator=g, device="cuda")
    q, k, v, grad = make(n).half(), make(n).half(), (make(n) * 4.0).half(), (make(n) * 2.0 ** -12).half()
    q2, k2, v2, grad2 = (make(other).half() for _ in range(4))
    causal = mate == "unseen"
    if mate == "nan":
        grad2[3], v2[5] = math.nan, math.nan
    elif mate == "inf":
        grad2[3], v2[5] = math.inf, -math.inf
    elif mate == "large":
        grad2[3], v2[5] = 6e4, 6e4
    elif mate == "no keys":
        k2, v2, grad2[:100], grad2[100:] = k2[:0], v2[:0], 6e4, math.nan
    elif mate == "no queries":
        q2, grad2, v2[:100], v2[100:] = q2[:0], grad2[:0], 6e4, math.inf
    elif mate == "unseen":
        grad2[:100], grad2[100:] = 6e4, math.nan
        k2, v2 = k2[:0], v2[:0]
    order = (lambda a, b: [b, a]) if first or causal else (lambda a, b: [a, b])
    leaves = [torch.cat(order(a, b)).requires_grad_() for a, b in ((q, q2), (k, k2), (v, v2))]
    if causal:                               # the other queries stand before the sample's keys
        lengths, key_lengths = [n + other], [n]
    else:
        lengths, key_lengths = order(n, q2.shape[0]), order(n, k2.shape[0])
    out = sparse_attention(*leaves, ends(lengths), ends(key_lengths), causal=causal)
    got = torch.autograd.grad(out, leaves, torch.cat(order(grad, grad2)))
    want = gradients64(q, k, v, grad, causal)
    eps = torch.finfo(torch.float16).eps
    for name, a, b, whole in zip("qkv", got, want, (q2, k2, v2)):
        at = whole.shape[0] if order(0, 1)[0] == 1 else 0
        assert relative(a[at:at + n], b) < eps + small_step(b), (name, relative(a[at:at + n], b))
