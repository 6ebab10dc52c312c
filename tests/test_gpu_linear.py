"""Pointwise linear layer on the GPU against its definition in 64 bits: every type, activation and
both kernels, at odd, unaligned and tiny sizes, forward and backward.

Tolerances are a running bound: a sum of n fp32 products is off by at most n steps of 2^-23 of
the sum of magnitudes (a step, not half, since the tensor cores may truncate), an activation by
2^-20 of its argument, and each rounding to the feature dtype by half a step of the value.
"""
import pytest
import torch

from sparseconv import _native
from sparseconv.ops.linear import Activation, sparse_linear

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = [Activation.NONE, Activation.RELU, Activation.GELU, Activation.SILU]
TINY = 2.0 ** -24            # subnormals of fp16


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _forward_ref(x, w, b, r, act):
    """(value, bound before the last rounding, argument, its bound)."""
    x, w = x.double(), w.double()
    K = x.shape[1]
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = (K + 2) * 2.0 ** -23 * mag
    v, _ = _act(z, act)
    e = 1.13 * ez + 2.0 ** -20 * (z.abs() + ez)          # |act'| <= 1.13
    if r is not None:
        v = v + r.double()
        e = e + 2.0 ** -23 * (v.abs() + r.double().abs())
    return v, e, z, ez


def _check(got, ref, bound, dtype, what):
    lim = bound + _half(dtype) * (ref.abs() + bound) + TINY
    bad = (got.double() - ref).abs() > lim
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                           f"{((got.double() - ref).abs() / lim).max():.3g} times")


def _inputs(M, Ci, Co, dtype, residual, bias=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s, k=1.0: (torch.randn(*s, generator=g, device="cuda") * k).to(dtype)
    return (mk(M, Ci), mk(Co, Ci, k=Ci ** -0.5), mk(Co) if bias else None, mk(M, Co) if residual else None, mk(M, Co))


# tensor-core sizes on and around tile edges, and sizes only the CUDA-core kernel takes
SIZES = [(1, 8, 8), (1, 256, 1024), (2, 64, 64), (17, 16, 24), (127, 64, 64), (128, 64, 256), (129, 72, 264),
         (300, 136, 40), (1000, 512, 520), (4097, 64, 256), (257, 1024, 136), (1, 3, 1), (5, 1, 7), (100, 35, 13),
         (259, 6, 32), (1000, 32, 13), (130, 257, 65), (33, 300, 200)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,Ci,Co", SIZES)
def test_forward(M, Ci, Co, dtype, act):
    x, w, b, r, _ = _inputs(M, Ci, Co, DT[dtype], residual=act != "gelu", bias=act != "silu")
    out = sparse_linear(x, w, b, residual=r, activation=act)
    v, e, _, _ = _forward_ref(x, w, b, r, act)
    _check(out, v, e, DT[dtype], "out")


def _backward_ref(x, w, b, g, act, dtype):
    """Gradients of feats, weight, bias with their bounds; dz enters the products rounded, its
    slope taken at the rounded argument (|act''| <= 0.8)."""
    _, _, z, ez = _forward_ref(x, w, b, None, act)
    _, slope = _act(z, act)
    gd = g.double()
    dz = gd * slope
    if act == "none":
        es = torch.zeros_like(dz)
    else:
        shift = ez + _half(dtype) * (z.abs() + ez) + TINY
        es = 0.8 * shift + 2.0 ** -20
        if act == "relu":                    # the kink can lie between the two arguments
            es = (z.abs() <= shift).double()
    e_sum = gd.abs() * es                    # dz before its rounding, as the bias sums take it
    e_dz = e_sum + (0.0 if act == "none" else _half(dtype) * (dz.abs() + e_sum) + TINY)
    xd, wd = x.double(), w.double()
    M, Co = dz.shape
    mag = dz.abs() + e_dz
    gx = (dz @ wd, e_dz @ wd.abs() + (Co + 2) * 2.0 ** -23 * (mag @ wd.abs()))
    gw = (dz.t() @ xd, e_dz.t() @ xd.abs() + (M + 2) * 2.0 ** -23 * (mag.t() @ xd.abs()))
    gb = (dz.sum(0), e_sum.sum(0) + (M + 2) * 2.0 ** -23 * (dz.abs() + e_sum).sum(0))
    return gx, gw, gb


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,Ci,Co", [(1, 8, 8), (3, 64, 128), (128, 64, 64), (200, 24, 72), (1000, 128, 256),
                                     (5000, 64, 256), (700, 264, 136), (2, 3, 5), (333, 35, 13), (4096, 32, 13),
                                     (777, 6, 33)])
def test_backward(M, Ci, Co, dtype, act):
    x, w, b, r, g = _inputs(M, Ci, Co, DT[dtype], residual=True, seed=1)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    out = sparse_linear(x, w, b, residual=r, activation=act)
    gx, gw, gb, gr = torch.autograd.grad(out, leaves, g)
    x, w, b = x.detach(), w.detach(), b.detach()
    for got, ref, what in zip((gx, gw, gb), _backward_ref(x, w, b, g, act, DT[dtype]), ("feats", "weight", "bias")):
        assert got.dtype == DT[dtype]
        _check(got, *ref, DT[dtype], what)
    assert torch.equal(gr, g)


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gradient_against_differences(act):
    """Directional derivatives of the fp32 layer against central differences of the 64-bit one."""
    x, w, b, _, g = _inputs(40, 24, 16, torch.float32, residual=False, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(sparse_linear(x, w, b, activation=act), leaves, g)
    f = lambda x, w, b: (_act(x @ w.t() + b, act)[0] * g.double()).sum()
    at = [t.detach().double() for t in leaves]
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i in range(3):
        d = torch.randn(at[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-4
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate(at)] for s in (1, -1))
        diff = (f(*up) - f(*down)) / (2 * h)
        # the difference is off by h^2 times a third derivative of order one per term; fp32 sums
        # by (K + M) steps of their magnitudes
        lim = ((grads[i].double() * d).abs().sum() + 1) * 1e-5
        assert abs((grads[i].double() * d).sum() - diff) < lim


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_views_that_start_anywhere(dtype, offset):
    """Contiguous views whose first element is not aligned to 16 bytes."""
    M, Ci, Co = 150, 64, 72
    t = DT[dtype]
    x0, w0, b0, r0, g0 = _inputs(M, Ci, Co, t, residual=True, seed=4)

    def shifted(a):
        buf = torch.empty(a.numel() + offset, dtype=t, device="cuda")
        v = buf[offset:].view(a.shape)
        v.copy_(a)
        return v
    x, w, b, r, g = (shifted(a) for a in (x0, w0, b0, r0, g0))
    v, e, _, _ = _forward_ref(x, w, b, r, "gelu")
    leaves = [a.requires_grad_(True) for a in (x, w, b)]
    out = sparse_linear(x, w, b, residual=r, activation="gelu")
    _check(out.detach(), v, e, t, "out")
    grads = torch.autograd.grad(out, leaves, g)
    for got, ref in zip(grads, _backward_ref(x0, w0, b0, g0, "gelu", t)):
        _check(got, *ref, t, "gradient")


def test_mixed_parameter_types():
    """fp32 master parameters with 16-bit features: cast for the product, gradients in fp32."""
    x, w, b, _, g = _inputs(500, 64, 48, torch.bfloat16, residual=False, seed=5)
    w32, b32 = w.float().requires_grad_(True), b.float().requires_grad_(True)
    out = sparse_linear(x, w32, b32, activation="silu")
    gw, gb = torch.autograd.grad(out, [w32, b32], g)
    assert out.dtype == torch.bfloat16 and gw.dtype == gb.dtype == torch.float32
    _, rw, rb = _backward_ref(x, w, b, g, "silu", torch.bfloat16)
    _check(gw, *rw, torch.float32, "weight")
    _check(gb, *rb, torch.float32, "bias")


def test_only_the_wanted_gradients():
    x, w, b, r, g = _inputs(300, 32, 48, torch.float16, residual=True, seed=6)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = torch.autograd.grad(sparse_linear(*full, residual=r, activation="gelu"), full, g)
    for i in range(3):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got = torch.autograd.grad(sparse_linear(*part, residual=r, activation="gelu"), part[i], g)[0]
        assert torch.equal(got, ref[i])
    r.requires_grad_(True)
    assert torch.equal(torch.autograd.grad(sparse_linear(x, w, b, residual=r, activation="gelu"), r, g)[0], g)


def test_expanded_output_gradient():
    x, w, b, _, _ = _inputs(70, 16, 24, torch.float32, residual=False)
    x.requires_grad_(True)
    sparse_linear(x, w, b).sum().backward()          # a gradient of stride zero
    ref = w.double().sum(0).expand(70, 16)
    _check(x.grad, ref, 26 * 2.0 ** -23 * w.double().abs().sum(0).expand(70, 16), torch.float32, "feats")


@pytest.mark.parametrize("dtype", list(DT))
def test_no_rows(dtype):
    x, w, b, r, g = _inputs(0, 16, 24, DT[dtype], residual=True)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    out = sparse_linear(x, w, b, residual=r, activation="gelu")
    assert out.shape == (0, 24)
    grads = torch.autograd.grad(out, leaves, g)
    assert grads[0].shape == (0, 16) and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ACTS)
def test_not_finite_values_stay_in_their_rows(dtype, act):
    x, w, b, _, _ = _inputs(300, 64, 64, DT[dtype], residual=False, seed=7)
    clean = sparse_linear(x, w, b, activation=act)
    x[5, 3], x[131, 0] = float("nan"), float("inf")
    out = sparse_linear(x, w, b, activation=act)
    rows = torch.ones(300, dtype=torch.bool, device="cuda")
    rows[[5, 131]] = False
    assert torch.equal(out[rows], clean[rows])
    assert out[5].isnan().all()
    if act in ("none", "relu"):
        assert (out[131].isinf() | (out[131] == 0)).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_same_bits_every_run(dtype):
    x, w, b, r, g = _inputs(20000, 64, 64, DT[dtype], residual=True, seed=8)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def once():
        out = sparse_linear(x, w, b, residual=r, activation="gelu")
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


def test_captured_and_replayed_step():
    x, w, b, r, g = _inputs(1000, 64, 128, torch.bfloat16, residual=True, seed=9)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        out = sparse_linear(x, w, b, residual=r, activation="silu")
        return [*torch.autograd.grad(out, leaves, g), out.detach()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    new = _inputs(1000, 64, 128, torch.bfloat16, residual=True, seed=10)
    with torch.no_grad():
        for t, s in zip((x, w, b, r, g), new):
            t.copy_(s)
    graph.replay()
    torch.cuda.synchronize()
    eager = step()
    assert all(torch.equal(a, c) for a, c in zip(held, eager))


def test_two_streams_at_once():
    a = _inputs(30000, 64, 128, torch.bfloat16, residual=True, seed=11)
    c = _inputs(30000, 64, 128, torch.bfloat16, residual=True, seed=12)
    want = [sparse_linear(t[0], t[1], t[2], residual=t[3], activation="gelu") for t in (a, c)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, t) in enumerate(zip(streams, (a, c))):
            with torch.cuda.stream(s):
                got[i].append(sparse_linear(t[0], t[1], t[2], residual=t[3], activation="gelu"))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)


def test_forced_kernels_agree_with_the_definition():
    x, w, b, r, _ = _inputs(513, 64, 96, torch.float16, residual=True, seed=13)
    v, e, _, _ = _forward_ref(x, w, b, r, "gelu")
    out, _ = _native.linear_forward(x, w, b, r, "gelu", kernel=_native.KERNEL_SIMT)
    _check(out, v, e, torch.float16, "CUDA cores")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,Ci,Co", [(37888, 64, 64), (40001, 128, 128), (38000, 8, 8), (41000, 72, 96), (50003, 64, 256),
                                     (38001, 24, 136), (39000, 128, 16), (37900, 16, 200), (60000, 128, 64)])
def test_backward_in_one_pass(M, Ci, Co, dtype, act):
    x, w, b, _, g = _inputs(M, Ci, Co, DT[dtype], residual=False, seed=21)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(sparse_linear(x, w, b, activation=act), leaves, g)
    x, w, b = x.detach(), w.detach(), b.detach()
    refs = _backward_ref(x, w, b, g, act, DT[dtype])
    for got, ref, what in zip(grads, refs, ("feats", "weight", "bias")):
        _check(got, *ref, DT[dtype], what)
    for i in range(3):                       # one gradient at a time: the same bits
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got = torch.autograd.grad(sparse_linear(*part, activation=act), part[i], g)[0]
        assert torch.equal(got, grads[i])


def test_backward_in_one_pass_same_bits_every_run():
    x, w, b, _, g = _inputs(70001, 128, 128, torch.bfloat16, residual=False, seed=22)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    once = lambda: torch.autograd.grad(sparse_linear(x, w, b, activation="gelu"), leaves, g)
    first = once()
    for _ in range(4):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


@pytest.mark.parametrize("M", [300, 40000])
def test_first_call_of_a_thread(M):
    """A thread that has made no CUDA call of its own (autograd runs backwards in such)."""
    import threading
    x, w, b, _, g = _inputs(M, 64, 64, torch.bfloat16, residual=False, seed=23)
    out, _ = _native.linear_forward(x, w, b, None, "none")
    want = _native.linear_backward(g, None, x, w, "none", torch.bfloat16, torch.bfloat16, (True, True, True))
    torch.cuda.synchronize()
    got = []

    def call():
        got.append(_native.linear_backward(g, None, x, w, "none", torch.bfloat16, torch.bfloat16, (True, True, True)))
        got.append(_native.linear_forward(x, w, b, None, "none")[0])
    t = threading.Thread(target=call)
    t.start()
    t.join()
    assert len(got) == 2
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got[0], want)) and torch.equal(got[1], out)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("act,residual", [("none", False), ("gelu", True)])
@pytest.mark.parametrize("M,Ci,Co", [(20000, 512, 520), (19001, 1024, 264), (9473, 520, 1032), (10000, 648, 512)])
def test_tiles_over_two_sms(M, Ci, Co, dtype, act, residual):
    """Many rows and channels: pairs of CTAs, with ragged last tiles in both directions."""
    x, w, b, r, g = _inputs(M, Ci, Co, DT[dtype], residual=residual, seed=31)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    out = sparse_linear(x, w, b, residual=r, activation=act)
    grads = torch.autograd.grad(out, leaves, g)
    x, w, b = x.detach(), w.detach(), b.detach()
    v, e, _, _ = _forward_ref(x, w, b, r, act)
    _check(out.detach(), v, e, DT[dtype], "out")
    for got, ref, what in zip(grads, _backward_ref(x, w, b, g, act, DT[dtype]), ("feats", "weight", "bias")):
        _check(got, *ref, DT[dtype], what)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("act,residual", [("none", True), ("gelu", False), ("silu", True)])
@pytest.mark.parametrize("M,Ci,Co", [(20000, 257, 131), (9001, 300, 203), (40001, 129, 72), (60000, 72, 93), (15000, 1001, 517),
                                     (200001, 129, 72)])
def test_channels_no_multiple_of_eight(M, Ci, Co, dtype, act, residual):
    """Around the row counts from which the copies into whole rows pay, forward and backward."""
    x, w, b, r, g = _inputs(M, Ci, Co, DT[dtype], residual=residual, bias=act != "silu", seed=41)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    out = sparse_linear(x, w, b, residual=r, activation=act)
    grads = torch.autograd.grad(out, leaves, g)
    x, w, b = (None if t is None else t.detach() for t in (x, w, b))
    v, e, _, _ = _forward_ref(x, w, b, r, act)
    _check(out.detach(), v, e, DT[dtype], "out")
    for got, ref, what in zip(grads, _backward_ref(x, w, b, g, act, DT[dtype]), ("feats", "weight", "bias")):
        _check(got, *ref, DT[dtype], what)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_bias_of_more_columns_than_shared_memory_keeps(dtype):
    x, w, b, r, _ = _inputs(200, 64, 5000, DT[dtype], residual=True, seed=51)
    v, e, _, _ = _forward_ref(x, w, b, r, "relu")
    _check(sparse_linear(x, w, b, residual=r, activation="relu"), v, e, DT[dtype], "out")


def test_more_than_2_to_31_elements():
    """The last rows of a large call equal the same rows alone (elements beyond a 32-bit index)."""
    M, Ci, Co = 1_100_003, 8, 2048
    x, w, b, _, _ = _inputs(M, Ci, Co, torch.bfloat16, residual=False, seed=52)
    out = sparse_linear(x, w, b, activation="relu")
    assert torch.equal(out[-1000:], sparse_linear(x[-1000:].clone(), w, b, activation="relu"))
    assert torch.equal(out[:1000], sparse_linear(x[:1000].clone(), w, b, activation="relu"))


def test_strided_parameters_and_second_derivatives():
    x, w, b, _, g = _inputs(300, 16, 24, torch.float32, residual=False, seed=53)
    want = sparse_linear(x, w, b)
    wide = torch.stack([w.t(), w.t()], -1)                       # [Ci, Co, 2]
    assert torch.equal(sparse_linear(x, wide[..., 0].t(), torch.stack([b, b], -1)[:, 0]), want)
    x.requires_grad_(True)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(sparse_linear(x, w, b), x, g, create_graph=True)
