"""Global gradient norm and clipping on the GPU against 64-bit sums: mixed types and sizes, views
that start anywhere, values whose squares leave fp32's range, values that are not finite.

The norm is a sum of eights in fp32 (8 half steps of 2^-24) added in fp64, so it is off by under
5 * 2^-24 of itself plus its rounding to fp32; the factor by a half step more, each product by a
half step, each output by its rounding.
"""
import pytest
import torch

from sparseconv.ops.clip import clip_grad_norm_, clip_gradients

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def _norm(grads):
    return sum((g.double() ** 2).sum() for g in grads).sqrt()


def _check(grads, outs, total, max_norm, want=None):
    want = _norm(grads) if want is None else want
    assert total.dtype == torch.float32 and total.dim() == 0
    assert abs(total.double() - want) <= 8 * U * want + 1e-45
    coef = min(1.0, max_norm / (float(want) + 1e-6))
    for g, o in zip(grads, outs):
        ref = g.double() * coef
        half = torch.finfo(g.dtype).eps / 2
        lim = (half + 16 * U) * ref.abs() + (2.0 ** -24 if g.dtype == torch.float16 else 1e-38)
        assert ((o.double() - ref).abs() <= lim).all()


def _grads(sizes, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=gen, device="cuda") * scale).to(DT[i % 3]) for i, s in enumerate(sizes)]


@pytest.mark.parametrize("sizes", [[1], [7], [8192], [8193], [0, 5, 0], [1, 2, 3, 4095, 100000, 8191, 16384],
                                   [64] * 63, [33] * 64, [17] * 65, [130] * 1100, [3_000_001, 5, 1_000_000]])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
def test_norm_and_scale(sizes, max_norm):
    grads = _grads(sizes)
    outs = [torch.full_like(g, 9.0) for g in grads]
    _check(grads, outs, clip_gradients(grads, max_norm, out=outs), max_norm)
    mine = [g.clone() for g in grads]
    total = clip_gradients(mine, max_norm)
    _check(grads, mine, total, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(mine, outs))


def test_in_place_below_the_limit_changes_nothing():
    grads = _grads([1000, 77, 40000])
    before = [g.clone() for g in grads]
    clip_gradients(grads, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("offset", [1, 2, 3, 4, 8])
def test_views_of_one_buffer(offset):
    """Gradients packed one after another, each starting wherever the last one ends."""
    buf = torch.randn(50000, device="cuda").to(torch.bfloat16)
    cuts = [offset, 1000 + offset, 1013 + offset, 30001 + offset, 49990]
    grads = [buf[a:b] for a, b in zip(cuts, cuts[1:])]
    keep = buf.clone()
    src = [g.clone() for g in grads]
    total = clip_gradients(grads, 1.0)
    _check(src, grads, total, 1.0)
    assert torch.equal(buf[:offset], keep[:offset]) and torch.equal(buf[49990:], keep[49990:])


@pytest.mark.parametrize("scale", [1e25, 1e18, 1e-18, 1e-25, 1e-30])
def test_squares_beyond_fp32(scale):
    grads = [torch.randn(3000, device="cuda") * scale, torch.randn(20, device="cuda") * scale]
    outs = [torch.empty_like(g) for g in grads]
    want = _norm(grads)
    total = clip_gradients(grads, 1.0, out=outs)
    assert abs(total.double() - want) <= 8 * U * want
    coef = min(1.0, 1.0 / (float(want) + 1e-6))
    for g, o in zip(grads, outs):       # a factor under 1e-38 would round in subnormal steps; none here does
        assert ((o.double() - g.double() * coef).abs() <= 16 * U * (g.double() * coef).abs() + 1e-38).all()


def test_zero_gradients():
    grads = [torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda", dtype=torch.float16)]
    assert clip_gradients(grads, 1.0).item() == 0.0
    assert not any(g.any() for g in grads)
    assert clip_gradients([torch.empty(0, device="cuda")], 1.0).item() == 0.0


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("norm_type", [2.0, float("inf")])
def test_not_finite(value, norm_type):
    grads = [torch.randn(5000, device="cuda"), torch.randn(100, device="cuda", dtype=torch.bfloat16)]
    grads[0][4321] = value
    ref = [g.clone() for g in grads]
    total = clip_gradients(grads, 1.0, norm_type)
    if value != value:
        assert total.isnan() and all(g.isnan().all() for g in grads)
    else:
        assert total.isinf()
        assert grads[0][4321].isnan() and not grads[1].any()
        assert torch.equal(grads[0].isnan(), ref[0].isinf())


def test_largest_magnitude():
    grads = _grads([1000, 77, 30000], seed=3)
    grads[1][5] = -50.0
    outs = [torch.empty_like(g) for g in grads]
    total = clip_gradients(grads, 2.0, float("inf"), out=outs)
    assert total.item() == 50.0
    _check(grads, outs, total, 2.0, want=torch.tensor(50.0, dtype=torch.float64, device="cuda"))


def test_permuted_memory():
    g = torch.randn(20, 30, 40, device="cuda").permute(2, 0, 1)
    ref = g.clone()
    total = clip_gradients([g], 1.0)
    _check([ref], [g], total, 1.0)


def test_parameters():
    lin = torch.nn.Linear(40, 30, device="cuda")
    other = torch.nn.Parameter(torch.randn(5, device="cuda"))
    (lin(torch.randn(10, 40, device="cuda")).square().sum() * 10).backward()
    grads = [p.grad.clone() for p in lin.parameters()]
    total = clip_grad_norm_([*lin.parameters(), other], 1.0)
    _check(grads, [p.grad for p in lin.parameters()], total, 1.0)
    assert clip_grad_norm_([other], 1.0).item() == 0.0


def test_refused_overlaps_leave_memory_alone():
    buf = torch.randn(300, device="cuda")
    keep = buf.clone()
    g = buf[:100]
    for grads, out in (([g, g], None), ([buf[:100], buf[50:150]], None), ([g], [buf[1:101]]),
                       ([buf[:100], buf[100:200]], [buf[100:200], buf[:100]]),
                       ([buf[:100], buf[200:300]], [buf[:100], buf[50:150]])):
        with pytest.raises(ValueError, match="overlap"):
            clip_gradients(grads, 0.1, out=out)
    torch.cuda.synchronize()
    assert torch.equal(buf, keep)
    # the same gradient read twice into separate outputs is no conflict
    outs = [torch.empty(100, device="cuda") for _ in range(2)]
    _check([g, g], outs, clip_gradients([g, g], 0.1, out=outs), 0.1)


def test_same_bits_every_run_and_replayed():
    grads = _grads([100000, 3, 777, 2_000_000], seed=5)
    outs = [torch.empty_like(g) for g in grads]
    total = clip_gradients(grads, 1.0, out=outs).clone()
    first = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_gradients(grads, 1.0, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = clip_gradients(grads, 1.0, out=outs)
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, total) and all(torch.equal(a, b) for a, b in zip(first, outs))
