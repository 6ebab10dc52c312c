"""A transformer block over voxels as a user writes it: norm, packed projections, rotary positions from the voxels'
coordinates, attention within each sample, output projection with the skip connection, a feed-forward pair, gradients and
clipping; against the block in 64 bits, captured into a graph, and its attention's waits at their limit.

fp32: sums of at most 4 C = 256 products a stage, ten stages each way, half a step of 2^-24 each: 256 * 10 * 6e-8 = 1.5e-4 of
the norm bounds it. bf16: some twenty roundings of 2^-9 on the way that add as independent errors, 2 sqrt(20) 2^-9 = 1.7e-2,
and for gradients, which pass them twice, 3.5e-2.
"""
import pytest
import torch

from sparseconv import SparseConvTensor, _native
from sparseconv.ops.attention import sparse_attention
from sparseconv.ops.clip import clip_gradients
from sparseconv.ops.linear import sparse_linear
from sparseconv.ops.norm import sparse_norm
from sparseconv.ops.rotary import rotary_steps, sparse_rotary

pytestmark = pytest.mark.gpu

C, B, H, D = 64, 3, 2, 32


def _setup(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    dense = torch.zeros(B, 12, 12, 12, C)
    occupied = torch.rand(B, 12, 12, 12, generator=g) < torch.tensor([0.3, 0.02, 0.15])[:, None, None, None]
    dense[occupied] = torch.randn(int(occupied.sum()), C, generator=g)
    x = SparseConvTensor.from_dense(dense.cuda().to(dtype))
    mk = lambda *s, k=1.0, o=0.0: (torch.randn(*s, generator=g) * k + o).cuda().to(dtype).requires_grad_(True)
    p = {"n1": mk(C, k=0.1, o=1.0), "qkv": mk(3 * C, C, k=C ** -0.5), "out": mk(C, C, k=C ** -0.5), "n2": mk(C, k=0.1, o=1.0),
         "up": mk(4 * C, C, k=C ** -0.5), "down": mk(C, 4 * C, k=(4 * C) ** -0.5)}
    return x, p


def _block(x, feats, p, offsets):
    qkv = sparse_linear(sparse_norm(feats, p["n1"], norm="rms"), p["qkv"]).view(-1, 3, H, D)
    q, k = sparse_rotary(qkv[:, 0], qkv[:, 1], x.indices[:, 1:])
    y = sparse_attention(q, k, qkv[:, 2], offsets).flatten(1)
    y = sparse_linear(y, p["out"], residual=feats)
    return sparse_linear(sparse_linear(sparse_norm(y, p["n2"], norm="rms"), p["up"], activation="gelu"), p["down"], residual=y)


def _block64(x, feats, p, offsets):
    f = torch.nn.functional
    rms = lambda t, w: t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt() * w
    qkv = f.linear(rms(feats, p["n1"]), p["qkv"]).view(-1, 3, H, D)
    theta = torch.tensor(rotary_steps(D // 6)[0], dtype=torch.float64, device=feats.device)
    angle = (x.indices[:, 1:].double()[:, :, None] * theta).flatten(1)[:, None]
    angle = f.pad(angle, (0, D // 2 - angle.shape[-1]))

    def turn(t):
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)
    q, k, v = turn(qkv[:, 0]), turn(qkv[:, 1]), qkv[:, 2]
    ends, parts = offsets.tolist(), []
    for i, j in zip(ends, ends[1:]):
        w = torch.softmax(torch.einsum("ihd,jhd->hij", q[i:j], k[i:j]) * D ** -0.5, -1)
        parts.append(torch.einsum("hij,jhd->ihd", w, v[i:j]))
    y = f.linear(torch.cat(parts).flatten(1), p["out"]) + feats
    return f.linear(f.gelu(f.linear(rms(y, p["n2"]), p["up"])), p["down"]) + y


def _near(got, ref, rel):
    assert (got.double() - ref).norm() <= rel * ref.norm(), ((got.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("dtype,forward,backward", [(torch.float32, 1.5e-4, 3e-4), (torch.bfloat16, 1.7e-2, 3.5e-2)])
def test_block(dtype, forward, backward):
    x, p = _setup(dtype)
    feats = x.features.detach().requires_grad_(True)
    offsets = x.batch_offsets()
    out = _block(x, feats, p, offsets)
    p64 = {k: t.detach().double().requires_grad_(True) for k, t in p.items()}
    feats64 = feats.detach().double().requires_grad_(True)
    ref = _block64(x, feats64, p64, offsets)
    _near(out.detach(), ref.detach(), forward)
    grad = torch.randn_like(out)
    grads = torch.autograd.grad(out, [feats, *p.values()], grad)
    refs = torch.autograd.grad(ref, [feats64, *p64.values()], grad.double())
    for got, want in zip(grads, refs):
        _near(got, want, backward)
    total = clip_gradients(list(grads[1:]), 1.0)
    _near(total, sum(t.square().sum() for t in refs[1:]).sqrt(), backward)


def test_block_in_a_graph():
    """Inference captured and replayed on new features; the gradients of a step captured beside it."""
    x, p = _setup(torch.bfloat16)
    offsets = x.batch_offsets()
    buffer = x.features.detach().clone()
    leaves = {k: t.detach().clone().requires_grad_(True) for k, t in p.items()}
    grad = torch.randn_like(buffer)
    with torch.no_grad():
        want = _block(x, buffer, p, offsets)
    want_grads = torch.autograd.grad(_block(x, buffer, leaves, offsets), list(leaves.values()), grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with torch.no_grad():
            out = _block(x, buffer, p, offsets)
        grads = torch.autograd.grad(_block(x, buffer, leaves, offsets), list(leaves.values()), grad)
    graph.replay()
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))
    other = torch.randn_like(buffer)
    with torch.no_grad():
        want = _block(x, other, p, offsets)
    buffer.copy_(other)
    graph.replay()
    assert torch.equal(out, want)
    assert _native.check_errors() == 0


def test_tokens_one_at_a_time_match_the_whole():
    """Causal attention over serialised voxels: the last query of a growing sample against the whole sample's rows."""
    q, k, v = (torch.randn(300, 4, 64, device="cuda").bfloat16() for _ in range(3))
    pos = torch.arange(300, device="cuda").int()
    rq, rk = sparse_rotary(q, k, pos)
    whole = sparse_attention(rq, rk, v, causal=True)
    for n in (1, 2, 64, 65, 129, 300):
        tq, _ = sparse_rotary(q[n - 1:n], None, pos[n - 1:n])
        off, key_off = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (1, n))
        one = sparse_attention(tq, rk[:n], v[:n], off, key_off, causal=True)
        # p is rounded against another running maximum, and sums are taken in another order: a rounding each
        assert (one.double() - whole[n - 1:n].double()).norm() <= 2.0 ** -7 * whole[n - 1:n].double().norm()


def _attention(n, H, K, D, what):
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, d = (torch.randn(n, h, D, generator=g, device="cuda").bfloat16() for h in (H, K, K, H))
    off = torch.tensor([0, n // 3, n], dtype=torch.int32, device="cuda")
    if what == "forward":
        return lambda: list(_native.attention_forward(q, k, v, off, off, False, 0.1, keep_stats=True)[:2])
    out, stats, args = _native.attention_forward(q, k, v, off, off, False, 0.1, keep_stats=True)
    needs = (True, False, False) if what == "query" else (False, True, True)
    return lambda: [t for t in _native.attention_backward_of(args, q, k, v, off, off, out, stats, d, needs) if t is not None]


@pytest.mark.parametrize("n,H,K,D,what", [(3000, 8, 8, 64, "forward"), (3000, 4, 2, 128, "forward"), (6000, 20, 20, 128, "forward"),
                                          (3000, 8, 8, 64, "query"), (3000, 4, 2, 128, "query"), (3000, 8, 8, 64, "key"), (3000, 4, 2, 128, "key")])
def test_wait_timeout_is_reported_and_the_context_stays_usable(n, H, K, D, what):
    call = _attention(n, H, K, D, what)
    ref = call()
    torch.cuda.synchronize()
    prev = _native.set_wait_limit_ns(1)
    try:
        with pytest.raises(RuntimeError, match="wait reached its time limit"):
            call()
            _native.check_errors()
    finally:
        _native.set_wait_limit_ns(prev)
    torch.cuda.synchronize()
    _native.reset_status()
    again = call()
    torch.cuda.synchronize()
    assert _native.check_errors() == 0
    assert all(torch.equal(a, b) for a, b in zip(again, ref))


def test_rows_past_32_bits_of_elements():
    """Keys and values whose elements pass 2^31 (a long cache): the last sample's keys lie behind them."""
    N, K, D = 4_200_000, 8, 64                                # 2.15e9 elements, 4.3 GB each
    k = torch.zeros(N, K, D, device="cuda", dtype=torch.float16)
    v = torch.zeros(N, K, D, device="cuda", dtype=torch.float16)
    m = 1000
    k[-m:], v[-m:] = torch.randn(m, K, D, device="cuda").half(), torch.randn(m, K, D, device="cuda").half()
    q = torch.randn(2, K, D, device="cuda").half()
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    key_off = torch.tensor([0, N - m, N], dtype=torch.int32, device="cuda")
    out = sparse_attention(q, k, v, off, key_off)
    alone = sparse_attention(q[1:], k[-m:].clone(), v[-m:].clone())
    assert (out[0] == 0).all()
    # the same keys, cut into other splits: sums in another order, p rounded against other maxima
    assert (out[1:].double() - alone.double()).norm() <= 2.0 ** -10 * alone.double().norm()
    pos = torch.zeros(N, dtype=torch.int32, device="cuda")
    pos[-1] = 7
    turned, _ = sparse_rotary(None, k, pos)[1], None
    assert torch.equal(turned[-2], k[-2]) and torch.equal(turned[-1:], sparse_rotary(k[-1:], None, pos[-1:])[0])
