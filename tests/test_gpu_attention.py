"""Attention against softmax in 64 bits, sample by sample; gradients against its autograd and against differences."""
import math

import pytest
import torch

from sparseconv import _native
from sparseconv.ops.attention import sparse_attention

pytestmark = pytest.mark.gpu


def ends(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def reference(q, k, v, lengths, key_lengths, causal, scale, grad=None):
    """(out, gradients) in 64 bits, and the sizes that the tolerances go by: sums of magnitudes."""
    H, K = q.shape[1], k.shape[1]
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    outs, i0, j0 = [], 0, 0
    for n, m in zip(lengths, key_lengths):
        a, b, c = leaves[0][i0:i0 + n], leaves[1][j0:j0 + m], leaves[2][j0:j0 + m]
        b, c = (torch.repeat_interleave(t, H // K, dim=1).transpose(0, 1) for t in (b, c))
        s = a.transpose(0, 1) @ b.transpose(1, 2) * scale
        hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
        if causal:
            hidden = torch.ones_like(hidden).triu(m - n + 1)
        s = s.masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1).masked_fill(hidden.all(1)[:, None], 0.0) if m else s
        outs.append((p @ c).transpose(0, 1))
        i0, j0 = i0 + n, j0 + m
    out = torch.cat(outs)
    grads = torch.autograd.grad(out, leaves, grad.double(), allow_unused=True) if grad is not None else ()
    return out.detach(), [torch.zeros_like(t) if g is None else g for t, g in zip(leaves, grads)]


def relative(got, want):
    norm = want.norm().item()
    return ((got.double() - want).norm().item() / norm) if norm else got.double().norm().item()


def tolerance(dtype):
    """Of the norm. A result's own rounding is eps / 2 at most (0.58 of it in the mean square); p, ds and out (in
    delta) are rounded as well, each within eps / 2 of the terms they enter: with terms of mixed signs the three add as
    independent errors to the result's own, at most four roundings. fp32: scores to 2^-24 of sqrt(D) |q| |k|, which the
    exponential turns into relative errors of p of a few 2^-22, and sums of up to a few thousand terms."""
    return {torch.float32: 4e-6}.get(dtype, 2.0 * torch.finfo(dtype).eps)


def run(lengths, key_lengths, H, K, D, dtype, causal=False, scale=None, seed=0, kernel=None, train=True):
    g = torch.Generator(device="cuda").manual_seed(seed + D)
    M, N = sum(lengths), sum(key_lengths)
    q, k, v = (torch.randn(r, h, D, generator=g, device="cuda").to(dtype).requires_grad_(train) for r, h in ((M, H), (N, K), (N, K)))
    grad = torch.randn(M, H, D, generator=g, device="cuda").to(dtype)
    out = sparse_attention(q, k, v, ends(lengths), ends(key_lengths), causal=causal, scale=scale)
    want, want_grads = reference(q, k, v, lengths, key_lengths, causal, D ** -0.5 if scale is None else scale, grad if train else None)
    assert out.dtype == dtype and out.shape == (M, H, D) and out.is_contiguous()
    assert relative(out.detach(), want) < tolerance(dtype)
    if train:
        for name, got, ref in zip("qkv", torch.autograd.grad(out, (q, k, v), grad), want_grads):
            assert got.shape == ref.shape and got.dtype == dtype
            assert relative(got, ref) < tolerance(dtype), (name, relative(got, ref))
    return out


TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 8, 16, 24, 33, 40, 64, 72, 96, 128])
def test_head_sizes(dtype, D):
    run([70, 129, 300], [70, 129, 300], 2, 2, D, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [136, 200, 256])
def test_wide_heads(dtype, D):
    run([40, 65], [90, 33], 2, 1, D, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m", [(1, 1), (1, 2), (2, 1), (1, 129), (127, 128), (128, 127), (129, 1), (255, 257), (256, 256), (257, 513),
                                 (1, 1000), (640, 15), (16, 16), (17, 31)])
def test_lengths(dtype, n, m):
    run([n], [m], 2, 2, 32, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,K", [(1, 1), (2, 1), (3, 1), (4, 2), (6, 2), (8, 1), (12, 4), (16, 16), (130, 1), (128, 1), (5, 5)])
def test_heads(dtype, H, K):
    run([37, 150], [90, 131], H, K, 16, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,K", [(2, 2), (8, 2), (6, 1)])
@pytest.mark.parametrize("lengths,key_lengths", [
    ([1, 300, 0, 129], [1, 300, 0, 129]),
    ([1, 1, 1], [500, 1, 130]),              # a new token each
    ([200, 130], [90, 128]),                 # queries before the first key see nothing
    ([129, 5], [400, 0]),
])
def test_causal(dtype, D, H, K, lengths, key_lengths):
    run(lengths, key_lengths, H, K, D, dtype, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_see_nothing(dtype):
    out = run([5, 140, 3], [7, 0, 64], 4, 2, 64, dtype)
    assert (out[5:145] == 0).all()
    out = run([200], [80], 2, 2, 64, dtype, causal=True)
    assert (out[:120] == 0).all() and (out[120:] != 0).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_many_short_samples(dtype):
    lengths = [(i * 37) % 71 for i in range(300)]
    run(lengths, lengths, 2, 2, 32, dtype)
    run([1] * 257, [(i * 13) % 40 for i in range(257)], 4, 1, 64, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "ends", "one"])
def test_many_samples_of_very_different_lengths(dtype, order):
    """A tile's sample is not where it would be if all were alike: before it, behind it, among empty ones."""
    lengths = {"up": [i // 2 for i in range(300)], "down": [i // 2 for i in range(300)][::-1],
               "ends": [900] + [0] * 200 + [1, 2] * 40 + [700], "one": [0] * 150 + [1000] + [0] * 33}[order]
    run(lengths, lengths, 4, 2, 32, dtype)
    run(lengths, lengths[::-1], 2, 2, 32, dtype, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_long_samples(dtype, D, causal):
    """Enough rows for two tiles of 128 queries a block, the last one with one tile or a part of it."""
    run([1500, 0, 1100, 1291], [1500, 0, 1100, 1291], 20, 10, D, dtype, causal=causal)
    run([1025, 1153], [700, 2000], 20, 20, D, dtype, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_few_queries_many_keys(dtype):
    """Keys in splits, joined."""
    run([1, 2, 1], [5000, 17, 9001], 8, 1, 64, dtype)
    run([3], [20011], 2, 2, 128, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_few_keys_many_queries(dtype):
    """Queries in splits for the keys' gradients."""
    run([7001, 3000], [3, 77], 4, 2, 64, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_key_has_no_score_gradient(dtype):
    """Its probability is 1 whatever the score: exactly no gradient."""
    q, k, v = (torch.randn(3, 2, 64, device="cuda").to(dtype).requires_grad_() for _ in range(3))
    out = sparse_attention(q, k, v, ends([1, 1, 1]))
    gq, gk, gv = torch.autograd.grad(out, (q, k, v), torch.randn_like(out))
    assert torch.equal(out, v) and (gq == 0).all() and (gk == 0).all() and (gv != 0).any()
    q, k, v = (torch.randn(200, 2, 64, device="cuda").to(dtype).requires_grad_() for _ in range(3))
    gq, _, _ = torch.autograd.grad(sparse_attention(q, k, v, causal=True), (q, k, v), torch.randn_like(q))
    assert (gq[0] == 0).all() and (gq[1] != 0).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [33, 64, 128, 136])
@pytest.mark.parametrize("m", [2, 3, 16])
def test_few_keys_keep_their_digits(dtype, D, m):
    """ds is a difference of grad . v and grad . out: with few keys out's rounding would be as large as any. With it out of the
    way, p's (in out and in the values' gradient), ds's and the result's roundings are left, 0.42 half steps each in the mean
    square of a uniform mantissa: at most sqrt(3) of them, under one half step."""
    lengths = [m] * 200
    g = torch.Generator(device="cuda").manual_seed(D + m)
    q, k, v, grad = (torch.randn(200 * m, 2, D, generator=g, device="cuda").to(dtype) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(sparse_attention(*leaves, ends(lengths)), leaves, grad)
    _, want = reference(*leaves, lengths, lengths, False, D ** -0.5, grad)
    for name, a, b in zip("qkv", got, want):
        assert relative(a, b) < torch.finfo(dtype).eps / 2, (name, relative(a, b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 10])
@pytest.mark.parametrize("n,D", [(40, 64), (3000, 64), (700, 128), (90, 33)])
def test_gradients_of_any_size(dtype, size, n, D):
    """Gradients far from 1 at rows of thousands of keys: ds is p times them, which fp16 could not hold as it is. The values' scale
    brings the results back to where fp16 holds them."""
    g = torch.Generator(device="cuda").manual_seed(n + D)
    q, k, v, grad = (torch.randn(n, 2, D, generator=g, device="cuda") for _ in range(4))
    leaves = [t.to(dtype).requires_grad_() for t in (q, k, v * (1.0 if size == 1.0 else 2.0 ** -4 if size > 1.0 else 64.0))]
    grad = (grad * size).to(dtype)
    got = torch.autograd.grad(sparse_attention(*leaves), leaves, grad)
    _, want = reference(*leaves, [n], [n], False, D ** -0.5, grad)
    for name, a, b in zip("qkv", got, want):
        # the results themselves: half of fp16's smallest step, over a result's root mean square
        small = 2.0 ** -25 / (b.norm().item() / b.numel() ** 0.5) if dtype == torch.float16 else 0.0
        assert relative(a, b) < tolerance(dtype) / 2 + small, (name, relative(a, b))


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_and_growing_scores(dtype):
    """Scores that rise along the keys, so that the running maximum changes in every tile, and large ones."""
    n, D = 700, 64
    q = torch.ones(n, 1, D, device="cuda").to(dtype)
    k = (torch.linspace(-40.0, 60.0, n, device="cuda")[:, None, None] * torch.ones(1, 1, D, device="cuda") / 8).to(dtype)
    v = torch.randn(n, 1, D, device="cuda").to(dtype)
    out = sparse_attention(q, k, v)
    want, _ = reference(q, k, v, [n], [n], False, D ** -0.5)
    # one rounding of p and of the result; in fp32, exponents of up to 690 are good to 690 * 2^-23
    assert relative(out, want) < max(tolerance(dtype), 3e-4 if dtype == torch.float32 else 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_whole_numbers_are_exact(dtype):
    """Equal scores: p = 2^-k for 2^k keys, and sums of small whole numbers are exact in fp32 and in the result."""
    v = torch.randint(-4, 5, (256, 2, 64), device="cuda").to(dtype).requires_grad_()
    q = torch.zeros(256, 2, 64, device="cuda").to(dtype)
    k = torch.randn(256, 2, 64, device="cuda").to(dtype)
    out = sparse_attention(q, k, v)
    want = (v.detach().double().sum(0, keepdim=True) / 256).to(dtype).expand_as(out)
    assert torch.equal(out.detach(), want)
    grad = torch.randint(-4, 5, out.shape, device="cuda").to(dtype)
    (gv,) = torch.autograd.grad(out, v, grad)
    assert torch.equal(gv, (grad.double().sum(0, keepdim=True) / 256).to(dtype).expand_as(gv))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,M,H", [(64, 4736, 64), (128, 4736, 64)])
def test_many_far_keys_keep_their_weight(dtype, D, M, H):
    """One key and 65,535 of e^-18 (2^-26) of its weight: together 1.0e-3 of the whole. There are tiles enough for no
    split, so all share one maximum. p of the far ones is 2^-19 where fp16 is lifted by 2^7, off by half of fp16's smallest step, 2^-25,
    and so by 2^-6 relative at most; in bf16, and the result's own rounding, by less than 2^-8 each."""
    n = 65536
    q = torch.zeros(M, H, D, device="cuda", dtype=dtype)
    k = torch.zeros(n, 1, D, device="cuda", dtype=dtype)
    v = torch.ones(n, 1, D, device="cuda", dtype=dtype)
    q[:, :, 0], k[1:, 0, 0], v[0] = 1.0, -18.0, 0.0
    far = (n - 1) * math.exp(-18.0)
    out = sparse_attention(q, k, v, scale=1.0).double()
    assert ((out / (far / (1.0 + far)) - 1.0).abs().max().item()) < 2.0 ** -6 + 2.0 ** -8 + 2.0 ** -8


@pytest.mark.parametrize("dtype", TYPES)
def test_other_samples_values_do_not_enter(dtype):
    """Infinities and NaN in the rows before and behind a sample, which its last tiles read."""
    for lengths, key_lengths in (([100, 75, 60], [100, 75, 60]), ([40, 33, 200], [90, 35, 128])):
        M, N = sum(lengths), sum(key_lengths)
        q, k, v, grad = (torch.randn(r, 2, 64, device="cuda").to(dtype) for r in (M, N, N, M))
        i0, i1, j0, j1 = lengths[0], lengths[0] + lengths[1], key_lengths[0], key_lengths[0] + key_lengths[1]
        for t, a, b in ((q, i0, i1), (grad, i0, i1), (k, j0, j1), (v, j0, j1)):
            t[:a], t[b:] = math.nan, math.inf
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        out = sparse_attention(q, k, v, ends(lengths), ends(key_lengths))
        gq, gk, gv = torch.autograd.grad(out, (q, k, v), grad)
        sub = [q.detach()[i0:i1], k.detach()[j0:j1], v.detach()[j0:j1]]
        want, grads = reference(*sub, [i1 - i0], [j1 - j0], False, 64 ** -0.5, grad[i0:i1])
        assert relative(out.detach()[i0:i1], want) < tolerance(dtype)
        for got, ref in zip((gq[i0:i1], gk[j0:j1], gv[j0:j1]), grads):
            assert relative(got, ref) < tolerance(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values_reach_their_rows_only(dtype):
    q, k, v = (torch.randn(300, 2, 64, device="cuda").to(dtype) for _ in range(3))
    clean = sparse_attention(q, k, v)
    q[7, 1, 3] = math.nan
    out = sparse_attention(q, k, v)
    assert out[7, 1].isnan().all()
    out[7, 1] = clean[7, 1]
    assert torch.equal(out, clean)
    k[200, 0, 0] = math.nan
    assert sparse_attention(q, k, v)[:, 0].isnan().all()


def test_strides():
    """Packed projections, heads first in memory, expanded heads, rows off 16-byte boundaries."""
    for dtype in TYPES:
        qkv = torch.randn(333, 3, 4, 64, device="cuda").to(dtype).requires_grad_()
        out = sparse_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], ends([133, 200]))
        grad = torch.randn_like(out)
        (got,) = torch.autograd.grad(out, qkv, grad)
        d = qkv.detach()
        want, grads = reference(d[:, 0], d[:, 1], d[:, 2], [133, 200], [133, 200], False, 0.125, grad)
        assert relative(out.detach(), want) < tolerance(dtype)
        assert relative(got, torch.stack(grads, 1)) < tolerance(dtype)
        same = sparse_attention(d[:, 0].contiguous(), d[:, 1].contiguous(), d[:, 2].contiguous(), ends([133, 200]))
        assert torch.equal(out.detach(), same)
        heads_first = d[:, 0].transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(sparse_attention(heads_first, d[:, 1], d[:, 2], ends([133, 200])), same)
        odd = torch.empty(333 * 256 + 1, device="cuda", dtype=dtype)[1:].view(333, 4, 64).copy_(d[:, 1])
        assert torch.equal(sparse_attention(d[:, 0], odd, d[:, 2], ends([133, 200])), same)
        spread = d[:, 1, :1].expand(333, 4, 64)
        assert torch.equal(sparse_attention(d[:, 0], spread, spread, ends([133, 200])),
                           sparse_attention(d[:, 0], spread[:, :1], spread[:, :1], ends([133, 200])))
        # a gradient with strides of zero
        leaf = d[:, 0].clone().requires_grad_()
        (a,) = torch.autograd.grad(sparse_attention(leaf, d[:, 1], d[:, 2]).sum(), leaf)
        (b,) = torch.autograd.grad(sparse_attention(leaf, d[:, 1], d[:, 2]), leaf, torch.ones_like(leaf))
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_run(dtype):
    q, k, v = (torch.randn(3000, 4, 64, device="cuda").to(dtype).requires_grad_() for _ in range(3))
    grad = torch.randn(3000, 4, 64, device="cuda").to(dtype)
    off = ends([1700, 0, 1300])

    def once():
        out = sparse_attention(q, k, v, off)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), grad)]
    first = once()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, once()))


@pytest.mark.parametrize("needs", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)])
def test_some_gradients(needs):
    q, k, v = (torch.randn(200, 2, 64, device="cuda").bfloat16() for _ in range(3))
    grad = torch.randn_like(q)
    every = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(sparse_attention(*every), every, grad)
    some = [t.clone().requires_grad_(bool(n)) for t, n in zip((q, k, v), needs)]
    got = torch.autograd.grad(sparse_attention(*some), [t for t in some if t.requires_grad], grad)
    assert all(torch.equal(g, w) for g, w in zip(got, [w for w, n in zip(want, needs) if n]))


def test_gradient_against_differences():
    q, k, v = (torch.randn(50, 2, 16, device="cuda", requires_grad=True) for _ in range(3))
    w = torch.randn(50, 2, 16, device="cuda")
    off = ends([20, 30])
    grads = torch.autograd.grad(sparse_attention(q, k, v, off, causal=True), (q, k, v), w)
    h = 2.0 ** -7
    for i, g in enumerate(grads):
        step = torch.randn(50, 2, 16, device="cuda")
        args = [t.detach().clone() for t in (q, k, v)]
        values = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * h * step
            values.append((sparse_attention(*moved, off, causal=True).double() * w.double()).sum().item())
        by_difference, by_gradient = (values[0] - values[1]) / (2 * h), (g.double() * step.double()).sum().item()
        # outputs to 2^-21 over 2 h each (root of 1,600 of them: 40), and the third derivative's h^2 / 6
        size = g.double().norm().item() * step.double().norm().item()
        assert abs(by_difference - by_gradient) < 40 * 2.0 ** -21 / h + size * h * h * 4


def test_nothing_given():
    q = torch.zeros(0, 2, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    k = torch.randn(5, 2, 64, device="cuda").half().requires_grad_()
    out = sparse_attention(q, k, k, ends([0]), ends([5]))
    gq, gk = torch.autograd.grad(out, (q, k), torch.zeros_like(out))
    assert out.shape == (0, 2, 64) and gq.shape == q.shape and (gk == 0).all()
    out = sparse_attention(k, q, q, ends([5]), ends([0]))
    gk, gq = torch.autograd.grad(out, (k, q), torch.ones_like(out))
    assert (out == 0).all() and (gk == 0).all() and gq.shape == q.shape


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [[0, 50, 40, 100], [1, 50, 60, 100], [0, 50, 60, 99], [0, 50, 60, 101], [-5, 50, 60, 100],
                                 [2 ** 31 - 1, -(2 ** 31), 7, 100], [0, 0, 0, 0]])
def test_bad_offsets_are_reported(dtype, bad):
    q = torch.randn(100, 2, 64, device="cuda").to(dtype).requires_grad_()
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    good = ends([50, 10, 40])
    for a, b in ((off, good), (good, off), (off, off)):
        with pytest.raises(RuntimeError, match="offsets"):
            sparse_attention(q, q, q, a, b)
            _native.check_errors()
    assert _native.check_errors() == 0


def test_streams_and_graphs():
    q, k, v = (torch.randn(500, 4, 64, device="cuda").bfloat16() for _ in range(3))
    pool = torch.randn(1, 4, 64, device="cuda").bfloat16()
    off, one = ends([500]), ends([1])
    want, pooled = sparse_attention(q, k, v, off), sparse_attention(pool, k, v, one, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [sparse_attention(q, k, v, off) for _ in range(3)]
    both = [sparse_attention(pool, k, v, one, off) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in other) and all(torch.equal(o, pooled) for o in both)
    graph = torch.cuda.CUDAGraph()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grad = torch.randn_like(q)
    eager = torch.autograd.grad(sparse_attention(*leaves, off), leaves, grad)
    with torch.cuda.graph(graph):
        a, b = sparse_attention(q, k, v, off), sparse_attention(pool, k, v, one, off)
        captured = torch.autograd.grad(sparse_attention(*leaves, off), leaves, grad)
    for _ in range(2):
        graph.replay()
    assert torch.equal(a, want) and torch.equal(b, pooled)
    assert all(torch.equal(x, y) for x, y in zip(captured, eager))


def test_one_tensor_as_all_inputs():
    x = torch.randn(200, 2, 32, device="cuda").bfloat16().requires_grad_()
    grad = torch.randn_like(x)
    (got,) = torch.autograd.grad(sparse_attention(x, x, x), x, grad)
    three = [x.detach().clone().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(sparse_attention(*three), three, grad)
    # autograd adds the parts in 16 bits: two roundings of the sum
    assert relative(got, sum(p.double() for p in parts)) < torch.finfo(torch.bfloat16).eps
