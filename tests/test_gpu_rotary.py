"""Rotary positions against the rotation in 64 bits, their gradient against the formula's and against differences."""
import math

import pytest
import torch

from sparseconv.ops.rotary import rotary_steps, sparse_rotary

pytestmark = pytest.mark.gpu


def reference(x, positions, layout, rotary_dim, steps, amplitude):
    """In 64 bits: pairs as complex numbers times amplitude * exp(i angle)."""
    x = x.detach().double()
    positions = positions[:, None] if positions.dim() == 1 else positions
    theta = torch.tensor(steps, dtype=torch.float64, device=x.device)
    angle = (positions.double()[:, :, None] * theta).flatten(1)[:, None]
    half, count = rotary_dim // 2, angle.shape[-1]
    head, rest = x[..., :rotary_dim], x[..., rotary_dim:]
    a, b = (head[..., :half], head[..., half:]) if layout == "half" else (head[..., 0::2], head[..., 1::2])
    turn = torch.polar(torch.full_like(angle, amplitude), angle)
    z = torch.complex(a.contiguous(), b.contiguous())
    z = torch.cat([z[..., :count] * turn, z[..., count:]], -1)
    parts = torch.cat([z.real, z.imag], -1) if layout == "half" else torch.stack([z.real, z.imag], -1).flatten(-2)
    return torch.cat([parts, rest], -1)


def check(got, want, dtype, amplitude):
    """One rounding of the result, and fp32's: sines to 2^-22, two products and a sum to 2^-23, of values that the pair's
    length bounds (the angle itself is exact to 2^-31 of a turn)."""
    assert got.dtype == dtype and got.is_contiguous()
    size = want.abs().amax().item() * amplitude if want.numel() else 0.0
    err = (got.double() - want).abs()
    bound = want.abs() * torch.finfo(dtype).eps / 2 + 2.0 * size * (2.0 ** -22 + 2.0 ** -23) + torch.finfo(dtype).tiny
    assert (err <= bound).all(), (err - bound).max().item()


CASES = [
    # rows, heads, key heads, size, rotary_dim, axes, layout, dtype
    (1, 1, 1, 2, 2, 1, "half", torch.float32),
    (1000, 8, 2, 64, 64, 3, "half", torch.bfloat16),
    (1000, 3, 3, 64, 64, 3, "interleaved", torch.float16),
    (777, 5, 1, 128, 96, 2, "half", torch.float16),
    (333, 2, 2, 35, 24, 3, "half", torch.float32),
    (333, 2, 2, 35, 24, 3, "interleaved", torch.float32),
    (257, 1, 1, 256, 256, 1, "half", torch.bfloat16),
    (63, 17, 1, 256, 250, 3, "interleaved", torch.float32),
    (129, 4, 2, 20, 12, 1, "half", torch.float16),
    (50, 300, 3, 8, 8, 2, "interleaved", torch.bfloat16),
    (4097, 1, 0, 17, 2, 1, "half", torch.bfloat16),
]


@pytest.mark.parametrize("rows,heads,key_heads,size,rotary_dim,axes,layout,dtype", CASES)
def test_matches_64_bits(rows, heads, key_heads, size, rotary_dim, axes, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + size)
    q = torch.randn(rows, heads, size, generator=g, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(rows, key_heads, size, generator=g, device="cuda").to(dtype).requires_grad_() if key_heads else None
    pos = torch.randint(-(1 << 31), (1 << 31) - 1, (rows, axes), generator=g, device="cuda").int()
    pos[: rows // 2] %= 512
    steps, amplitude = rotary_steps(rotary_dim // 2 // axes)
    rq, rk = sparse_rotary(q, k, pos, layout=layout, rotary_dim=rotary_dim)
    for t, r in ((q, rq), (k, rk)):
        if t is not None:
            check(r.detach(), reference(t, pos, layout, rotary_dim, steps, amplitude), dtype, amplitude)
    gq = torch.randn(rows, heads, size, generator=g, device="cuda").to(dtype)
    outs, grads, leaves = [rq], [gq], [q]
    if k is not None:
        outs, grads, leaves = [rq, rk], [gq, torch.randn(k.shape, generator=g, device="cuda").to(dtype)], [q, k]
    for got, grad in zip(torch.autograd.grad(outs, leaves, grads), grads):
        back = reference(grad, pos, layout, rotary_dim, [-s for s in steps], amplitude)
        check(got, back, dtype, amplitude)


def test_gradient_against_differences():
    """Linear in its input: a difference of outputs is the derivative but for roundings (fp32: 2^-22 of the values)."""
    q = torch.randn(40, 2, 24, device="cuda", requires_grad=True)
    pos = torch.randint(0, 100, (40, 3), device="cuda").int()
    w, step = torch.randn(40, 2, 24, device="cuda"), torch.randn(40, 2, 24, device="cuda")
    out, _ = sparse_rotary(q, None, pos, scaling="yarn", factor=2.0, trained_size=50)
    (grad,) = torch.autograd.grad(out, q, w)
    more, _ = sparse_rotary(q.detach() + step, None, pos, scaling="yarn", factor=2.0, trained_size=50)
    by_difference = ((more - out.detach()).double() * w.double()).sum()
    assert abs(by_difference - (grad.double() * step.double()).sum()) < 40 * 2 * 24 * 2.0 ** -20


@pytest.mark.parametrize("scaling,factor,trained", [("none", 1.0, None), ("linear", 3.0, None), ("ntk", 4.0, None), ("yarn", 4.0, 300)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scalings(scaling, factor, trained, layout):
    q = torch.randn(500, 4, 64, device="cuda").bfloat16()
    pos = torch.randint(0, 1 << 20, (500,), device="cuda").int()
    steps, amplitude = rotary_steps(32, 10000.0, scaling, factor, trained)
    out, none = sparse_rotary(q, None, pos, layout=layout, scaling=scaling, factor=factor, trained_size=trained)
    assert none is None
    check(out, reference(q, pos, layout, 64, steps, amplitude), torch.bfloat16, amplitude)


def test_far_positions_keep_their_angle():
    """fp32 angles would be off by 2^31 * 2^-24 = 128 radians."""
    pos = torch.tensor([2 ** 31 - 1, -(2 ** 31), 12345678, 0], device="cuda").int()
    q = torch.zeros(4, 1, 2, device="cuda")
    q[..., 0] = 1.0
    out, _ = sparse_rotary(q, None, pos)
    # in 64 bits the product is exact (step 1) and the cosine good to 2^-53
    for i, p in enumerate(pos.tolist()):
        # 2^31 steps of 2^-65 of a turn from rounding the step (2^-34 turns: 4e-10), and fp32's cosine
        assert abs(out[i, 0, 0].item() - math.cos(p)) < 4e-7 and abs(out[i, 0, 1].item() - math.sin(p)) < 4e-7


def test_strided_inputs_and_positions():
    """Views into packed projections, the coordinates' columns, heads that are not contiguous, misaligned rows."""
    qkv = torch.randn(200, 3, 4, 32, device="cuda").half()
    indices = torch.randint(0, 64, (200, 4), device="cuda").int()
    steps, amplitude = rotary_steps(5)
    q, k = sparse_rotary(qkv[:, 0], qkv[:, 1], indices[:, 1:])
    pos = indices[:, 1:].contiguous()
    check(q, reference(qkv[:, 0], pos, "half", 32, steps, amplitude), torch.float16, 1.0)
    check(k, reference(qkv[:, 1], pos, "half", 32, steps, amplitude), torch.float16, 1.0)
    odd = torch.randn(200, 4 * 32 + 1, device="cuda").half()[:, 1:].view(200, 4, 32)
    check(sparse_rotary(odd, None, indices[:, 1:])[0], reference(odd, pos, "half", 32, steps, amplitude), torch.float16, 1.0)
    turned = torch.randn(200, 32, 4, device="cuda").half().transpose(1, 2)
    check(sparse_rotary(turned, None, indices[:, 1:])[0], reference(turned, pos, "half", 32, steps, amplitude), torch.float16, 1.0)
    spread = torch.randn(200, 1, 32, device="cuda").half().expand(200, 4, 32)
    check(sparse_rotary(spread, None, indices[:, 1:])[0], reference(spread, pos, "half", 32, steps, amplitude), torch.float16, 1.0)


def test_nothing_to_turn():
    pos = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    q, k = sparse_rotary(torch.zeros(0, 2, 12, device="cuda"), torch.zeros(0, 1, 12, device="cuda"), pos)
    assert q.shape == (0, 2, 12) and k.shape == (0, 1, 12)


def test_special_values_stay_in_their_pair():
    q = torch.randn(64, 2, 16, device="cuda")
    q[3, 1, 2], q[5, 0, 7] = math.nan, math.inf
    pos = torch.arange(64, device="cuda").int()
    out, _ = sparse_rotary(q, None, pos)
    bad = ~torch.isfinite(out)
    assert bad[3, 1, 2] and bad[3, 1, 10] and (bad[5, 0, 7] or bad[5, 0, 15]) and bad.sum() <= 4


def test_only_one_gradient_asked():
    q = torch.randn(10, 2, 8, device="cuda", requires_grad=True)
    k = torch.randn(10, 1, 8, device="cuda", requires_grad=True)
    pos = torch.arange(10, device="cuda").int()
    a, b = sparse_rotary(q, k, pos)
    (gk,) = torch.autograd.grad(b.sum(), k)
    assert gk.shape == k.shape
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(sparse_rotary(q, k, pos)[0].sum(), q, create_graph=True)


def test_captured_and_on_another_stream():
    q = torch.randn(100, 2, 32, device="cuda").bfloat16()
    pos = torch.randint(0, 99, (100, 3), device="cuda").int()
    want, _ = sparse_rotary(q, None, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = sparse_rotary(q, None, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, _ = sparse_rotary(q, None, pos)
    graph.replay()
    assert torch.equal(other, want) and torch.equal(captured, want)
