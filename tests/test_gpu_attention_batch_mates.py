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


@pytest.mark.parametrize("mate", ["nan", "inf", "large", "no keys", "no queries", "unseen"])
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


TYPES16 = [torch.bfloat16, torch.float16]


def apart(rows, D, dtype, seed, heads=2):
    """Queries, keys, values and gradients whose scores are far apart, as a trained network's: a row's weight is on a few keys, and
    out's rounding then of ds's size, however many keys there are. What is left without it is four roundings (p's in out and in
    the values' gradient, ds's, the result's) of 0.42 half steps each in the mean square of a uniform mantissa: under one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, grad = (torch.randn(r, heads, D, generator=g, device="cuda") for r in rows)
    return [t.to(dtype).requires_grad_() for t in (q * 4.0, k, v)], grad.to(dtype)


def check(got, want, dtype):
    for name, a, b in zip("qkv", got, want):
        assert relative(a, b) < torch.finfo(dtype).eps / 2, (name, relative(a, b) / (torch.finfo(dtype).eps / 2))


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("D", [64, 128, 136])
def test_short_samples_beside_a_long_one(dtype, D):
    """Windows of two keys beside a scene of 20,000: as near to 64 bits, and to the bit, as without it."""
    m, windows, long = 2, 100, 20000
    leaves, grad = apart([windows * m + long] * 4, D, dtype, D)
    got = torch.autograd.grad(sparse_attention(*leaves, ends([m] * windows + [long])), leaves, grad)
    each = [gradients64(*(t.detach()[i:i + m] for t in leaves), grad[i:i + m]) for i in range(0, windows * m, m)]
    check([t[:windows * m] for t in got], [torch.cat(t) for t in zip(*each)], dtype)
    alone = [t.detach()[:windows * m].clone().requires_grad_() for t in leaves]
    want = torch.autograd.grad(sparse_attention(*alone, ends([m] * windows)), alone, grad[:windows * m])
    assert all(torch.equal(a[:windows * m], b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("D", [64, 128, 136])
def test_first_rows_of_a_long_causal_sample(dtype, D):
    """They see 1 to 16 keys."""
    leaves, grad = apart([2000] * 4, D, dtype, D)
    (gq,) = torch.autograd.grad(sparse_attention(*leaves, causal=True), leaves[:1], grad)
    check([gq[:16]], [gradients64(*leaves, grad, causal=True)[0][:16]], dtype)


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,m", [(300, 129), (300, 257), (700, 2000)])
def test_few_keys_that_count_among_many(dtype, D, n, m):
    leaves, grad = apart([n, m, m, n], D, dtype, m)
    got = torch.autograd.grad(sparse_attention(*leaves, ends([n]), ends([m])), leaves, grad)
    check(got, gradients64(*leaves, grad), dtype)
