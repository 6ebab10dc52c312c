"""The gated residual step with its norms on the GPU against its definition in 64 bits, forward
and backward, at every lane layout of the kernels, with samples of uneven and no size.

The reference carries a running bound along: each fp32 operation adds half a step (2^-24) of its
result, a sum of n terms n half steps of the sum of magnitudes.
"""
import pytest
import torch

from sparseconv import SparseConvTensor, _native
from sparseconv.ops.norm import Norm, sparse_norm, sparse_residual_norm

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
EPS = 1e-5


def _mean(v, e):
    C = v.shape[1]
    return v.mean(1, keepdim=True), e.mean(1, keepdim=True) + C * U * (v.abs() + e).mean(1, keepdim=True)


def _normalise(t, et, kind):
    """(normalised, bound, rstd, bound)"""
    if kind == "none":
        return t, et, torch.ones_like(t[:, :1]), torch.zeros_like(t[:, :1])
    if kind == "layer":
        m, em = _mean(t, et)
        t, et = t - m, et + em + U * (t.abs() + m.abs())
    q, eq = _mean(t * t, 2 * t.abs() * et + et * et + U * t * t)
    rstd = (q + EPS).rsqrt()
    low = (q + EPS - eq).clamp_min(EPS * 0.5)         # rsqrt is off most towards smaller arguments
    er = (low.rsqrt() - rstd) + 4 * U * rstd
    n = t * rstd
    return n, et * (rstd + er) + t.abs() * er + U * n.abs(), rstd, er


def _normalise_back(t, et, n, en, rstd, er, kind):
    if kind == "none":
        return t, et
    q, eq = _mean(t * n, et * n.abs() + t.abs() * en + et * en + U * (t * n).abs())
    s, es = _mean(t, et) if kind == "layer" else (torch.zeros_like(q), torch.zeros_like(q))
    o = t - s - n * q
    eo = et + es + n.abs() * eq + en * q.abs() + en * eq + 4 * U * (t.abs() + s.abs() + (n * q).abs())
    return o * rstd, eo * (rstd + er) + o.abs() * er + U * (o * rstd).abs()


def _ref(x, r, g, w1, b1, w2, b2, sample, alpha, norm, next_norm, dh=None, dy=None):
    """{name: (value, bound)} of the outputs, and of the gradients where dh or dy is given."""
    d = lambda t: None if t is None else t.double()
    x, r, dh, dy = d(x), d(r), d(dh), d(dy)

    def rows(p, default):
        if p is None:
            return torch.full_like(x[:1], default)
        p = p.double()
        return p[sample] if p.dim() == 2 else p[None]
    gr, w1r, b1r, w2r, b2r = rows(g, 1.0), rows(w1, 1.0), rows(b1, 0.0), rows(w2, 1.0), rows(b2, 0.0)
    zero = torch.zeros_like(x)
    n1, e1, rstd1, er1 = _normalise(x, zero, norm)
    u = n1 * w1r + b1r
    eu = e1 * w1r.abs() + 2 * U * ((n1 * w1r).abs() + u.abs())
    res = zero if r is None else alpha * r
    h = res + gr * u
    eh = gr.abs() * eu + 3 * U * (res.abs() + (gr * u).abs() + h.abs())
    out = {"hidden": (h, eh)}
    if next_norm != "none":
        n2, e2, rstd2, er2 = _normalise(h, eh, next_norm)
        y = n2 * w2r + b2r
        out["normed"] = (y, e2 * w2r.abs() + 2 * U * ((n2 * w2r).abs() + y.abs()))
    if dh is None and dy is None:
        return out
    G, eG = (zero, zero) if dh is None else (dh, zero)
    sums = {}
    if dy is not None:
        sums["next_bias"] = (dy, zero)
        sums["next_weight"] = (dy * n2, dy.abs() * e2 + U * (dy * n2).abs())
        t, et = _normalise_back(dy * w2r, U * (dy * w2r).abs(), n2, e2, rstd2, er2, next_norm)
        eG = eG + et + U * (G.abs() + t.abs())
        G = G + t
    out["residual"] = (alpha * G, abs(alpha) * eG + U * (alpha * G).abs())
    sums["gate"] = (G * u, eG * u.abs() + G.abs() * eu + eG * eu + U * (G * u).abs())
    du, edu = G * gr, eG * gr.abs() + U * (G * gr).abs()
    sums["bias"] = (du, edu)
    sums["weight"] = (du * n1, edu * n1.abs() + du.abs() * e1 + edu * e1 + U * (du * n1).abs())
    t, et = du * w1r, edu * w1r.abs() + U * (du * w1r).abs()
    out["feats"] = _normalise_back(t, et, n1, e1, rstd1, er1, norm)
    for name, p in (("gate", g), ("weight", w1), ("bias", b1), ("next_weight", w2), ("next_bias", b2)):
        if p is None:
            continue
        v, e = sums.get(name, (zero, zero))
        e = e + U * (x.shape[0] + 40) * (v.abs() + e)        # the sum's own half steps
        if p.dim() == 2:
            z = torch.zeros(p.shape, dtype=torch.float64, device=x.device)
            out[name] = z.index_add(0, sample, v), z.index_add(0, sample, e)
        else:
            out[name] = v.sum(0), e.sum(0)
    return out


def _check(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2
    lim = bound + half * (ref.abs() + bound) + 2.0 ** -24 * (got.dtype == torch.float16) + 1e-37
    bad = ~((got.double() - ref).abs() <= lim)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                           f"{((got.double() - ref).abs() / lim).max():.3g} times")


def _offsets(M, B, seed):
    """B samples, several of them empty (the first and the last too when there are enough)."""
    if B == 1:
        return torch.tensor([0, M], dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, M + 1, (B - 1,), generator=gen).sort().values
    if B >= 4:
        cuts[0], cuts[-1] = 0, M
    return torch.cat([torch.tensor([0]), cuts, torch.tensor([M])]).to(torch.int32).cuda()


def _case(M, C, B, dtype, ptype, gate, norm, next_norm, per_sample=(), residual=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s, k=1.0, o=0.0, t=dtype: (torch.randn(*s, generator=gen, device="cuda") * k + o).to(t)
    shape = lambda name: (B, C) if name in per_sample else (C,)
    p = dict(gate=None, weight=None, bias=None, next_weight=None, next_bias=None)
    if gate:
        p["gate"] = mk(*shape("gate"), k=0.5, t=ptype)
    if norm != "none":
        p["weight"] = mk(*shape("weight"), k=0.2, o=1.0, t=ptype)
        p["bias"] = mk(*shape("bias"), k=0.3, t=ptype) if norm == "layer" else None
    if next_norm != "none":
        p["next_weight"] = mk(*shape("next_weight"), k=0.2, o=1.0, t=ptype)
        p["next_bias"] = mk(*shape("next_bias"), k=0.3, t=ptype) if next_norm == "layer" else None
    x = mk(M, C, k=2.0, o=0.5)
    r = mk(M, C) if residual else None
    off = _offsets(M, B, seed)
    sample = torch.repeat_interleave(torch.arange(B, device="cuda"), (off[1:] - off[:-1]).long())
    return x, r, p, off, sample, mk(M, C), mk(M, C)


def _run(M, C, B, dtype, ptype, gate, norm, next_norm, per_sample=(), residual=True, alpha=1.0, use=(True, True), seed=0):
    x, r, p, off, sample, dh, dy = _case(M, C, B, dtype, ptype, gate, norm, next_norm, per_sample, residual, seed)
    leaves = {"feats": x, "residual": r, **p}
    leaves = {k: t.requires_grad_(True) for k, t in leaves.items() if t is not None}
    hidden, normed = sparse_residual_norm(x, r, batch_offsets=off, residual_scale=alpha, norm=norm,
                                          next_norm=next_norm, eps=EPS, **p)
    ref = _ref(x.detach(), None if r is None else r.detach(), *(None if t is None else t.detach() for t in p.values()),
               sample, alpha, norm, next_norm, dh if use[0] else None, dy if use[1] and next_norm != "none" else None)
    _check(hidden.detach(), *ref["hidden"], "hidden")
    if next_norm == "none":
        assert normed is None
    else:
        _check(normed.detach(), *ref["normed"], "normed")
    outs = [(hidden, dh)] * use[0] + [(normed, dy)] * (use[1] and next_norm != "none")
    if not outs:
        return
    grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs])
    for k, g in zip(leaves, grads):
        assert g.dtype == leaves[k].dtype and g.shape == leaves[k].shape
        _check(g, *ref[k], k)


# every lane layout: sub-warp, warp and block rows, eight columns at a time or single ones
CHANNELS = [1, 2, 3, 8, 16, 24, 35, 64, 100, 129, 200, 256, 264, 500, 512, 520, 1000, 1001, 1024, 1032, 2050, 4096, 8192]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", CHANNELS)
def test_every_layout(C, dtype):
    _run(131, C, 3, DT[dtype], torch.float32, True, "layer", "layer", per_sample=("gate",), seed=C)


@pytest.mark.parametrize("norm", ["none", "layer", "rms"])
@pytest.mark.parametrize("next_norm", ["none", "layer", "rms"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", [64, 35, 300])
def test_every_kind(C, dtype, norm, next_norm):
    _run(200, C, 4, DT[dtype], DT[dtype], True, norm, next_norm, seed=3)
    _run(65, C, 2, DT[dtype], torch.float32, False, norm, next_norm, residual=False, seed=4)


@pytest.mark.parametrize("M", [1, 2, 31, 1000, 20011])
@pytest.mark.parametrize("B", [1, 2, 7, 40])
def test_samples(M, B):
    """All five parameters with a row per sample; more samples than rows among them."""
    _run(M, 64, B, torch.bfloat16, torch.float32, True, "layer", "layer",
         per_sample=("gate", "weight", "bias", "next_weight", "next_bias"), seed=M + B)


@pytest.mark.parametrize("use", [(True, False), (False, True)])
@pytest.mark.parametrize("C", [64, 600])
def test_one_output_used(C, use):
    _run(300, C, 3, torch.float16, torch.float16, True, "rms", "layer", per_sample=("gate",), use=use, alpha=0.7, seed=5)


def test_many_rows():
    _run(300001, 32, 5, torch.float16, torch.float32, True, "layer", "rms", per_sample=("gate", "next_weight"), seed=6)


def test_gradient_against_differences():
    x, r, p, off, sample, dh, dy = _case(50, 24, 3, torch.float32, torch.float32, True, "layer", "rms", ("gate",), seed=7)
    leaves = [t.requires_grad_(True) for t in (x, r, *[t for t in p.values() if t is not None])]
    names = [k for k, t in p.items() if t is not None]
    hidden, normed = sparse_residual_norm(x, r, batch_offsets=off, norm="layer", next_norm="rms", eps=EPS, **p)
    grads = torch.autograd.grad([hidden, normed], leaves, [dh, dy])

    def f(x, r, *ps):
        q = dict(p, **dict(zip(names, ps)))
        o = _ref(x, r, *q.values(), sample, 1.0, "layer", "rms")
        return (o["hidden"][0] * dh.double()).sum() + (o["normed"][0] * dy.double()).sum()
    at = [t.detach().double() for t in leaves]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(len(at)):
        d = torch.randn(at[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate(at)] for s in (1, -1))
        got, want = (grads[i].double() * d).sum(), (f(*up) - f(*down)) / (2 * h)
        # h^2 of a third derivative of order (1 / deviation)^2, and the fp32 gradient's own steps
        assert abs(got - want) < 1e-5 * ((grads[i].double() * d).abs().sum() + 1)


@pytest.mark.parametrize("C", [64, 1024])
def test_large_common_offset(C):
    """Rows whose mean is a thousand times their deviation: the variance keeps its digits."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(40, C, generator=g, device="cuda") + 1000.0
    ref = torch.nn.functional.layer_norm(x.double(), (C,), eps=EPS)
    # the mean is off by C half steps of 1000, the deviations by that much
    assert (sparse_norm(x).double() - ref).abs().max() < 4 * C * U * 1000


def test_constant_and_zero_rows():
    x = torch.zeros(3, 64, device="cuda")
    x[1] = 7.0
    for kind in (Norm.LAYER, Norm.RMS):
        y = sparse_norm(x, norm=kind)
        assert torch.isfinite(y).all() and not y[0].any()
    assert not sparse_norm(x)[1].any()


def test_not_finite_values_stay_in_their_rows():
    x = torch.randn(100, 64, device="cuda", dtype=torch.bfloat16)
    clean = sparse_norm(x)
    x[3, 5], x[50, 0] = float("inf"), float("nan")
    y = sparse_norm(x)
    keep = torch.ones(100, dtype=torch.bool, device="cuda")
    keep[[3, 50]] = False
    assert torch.equal(y[keep], clean[keep]) and y[50].isnan().all()


@pytest.mark.parametrize("dtype", list(DT))
def test_no_rows(dtype):
    x, r, p, off, *_ = _case(0, 16, 1, DT[dtype], torch.float32, True, "layer", "layer", ())
    leaves = [t.requires_grad_(True) for t in (x, r, *[t for t in p.values() if t is not None])]
    hidden, normed = sparse_residual_norm(x, r, norm="layer", next_norm="layer", **p)
    grads = torch.autograd.grad([hidden, normed], leaves, [torch.zeros_like(hidden), torch.zeros_like(normed)])
    assert hidden.shape == normed.shape == (0, 16)
    assert all(not g.any() for g in grads)


def test_views_that_start_anywhere():
    x, r, p, off, sample, _, _ = _case(99, 64, 2, torch.float16, torch.float32, True, "layer", "layer", ("gate",))
    want = sparse_residual_norm(x, r, batch_offsets=off, norm="layer", next_norm="layer", **p)
    ref = _ref(x, r, *p.values(), sample, 1.0, "layer", "layer")
    buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    v = buf[1:].view(x.shape)
    v.copy_(x)
    got = sparse_residual_norm(v, r, batch_offsets=off, norm="layer", next_norm="layer", **p)
    for o in (got, want):
        _check(o[0], *ref["hidden"], "hidden")
        _check(o[1], *ref["normed"], "normed")


@pytest.mark.parametrize("bad", [[1, 50, 100], [0, 50, 99], [0, 70, 60], [0, 120, 100], [-5, 50, 100]])
def test_bad_offsets_raise(bad):
    x = torch.randn(100, 64, device="cuda")
    gate = torch.randn(2, 64, device="cuda")
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="sample offsets"):
        sparse_residual_norm(x, x, gate=gate, batch_offsets=off)
        _native.check_errors()
    _native.reset_status()
    sparse_residual_norm(x, x, gate=gate, batch_offsets=torch.tensor([0, 50, 100], dtype=torch.int32, device="cuda"))
    _native.check_errors()


def test_offsets_of_a_sparse_tensor():
    ind = torch.tensor([[0, 0, 0, 0], [0, 1, 0, 0], [2, 0, 0, 0], [2, 0, 0, 1], [2, 3, 0, 0]], dtype=torch.int32, device="cuda")
    t = SparseConvTensor(torch.randn(5, 16, device="cuda"), ind, [4, 4, 4], 4)
    off = t.batch_offsets()
    assert off.tolist() == [0, 2, 2, 5, 5] and off.dtype == torch.int32
    gate = torch.randn(4, 16, device="cuda")
    hidden, _ = sparse_residual_norm(t.features, t.features, gate=gate, batch_offsets=off, next_norm="none")
    assert torch.allclose(hidden, t.features * (1 + gate[[0, 0, 2, 2, 2]]), rtol=1e-6, atol=1e-6)


def test_same_bits_every_run_and_replayed():
    x, r, p, off, _, dh, dy = _case(30000, 64, 6, torch.bfloat16, torch.float32, True, "layer", "layer", ("gate",), seed=8)
    leaves = [t.requires_grad_(True) for t in (x, r, *[t for t in p.values() if t is not None])]

    def step():
        o = sparse_residual_norm(x, r, batch_offsets=off, norm="layer", next_norm="layer", **p)
        # detached: a live eager graph of the same leaves would break the capture of a backward
        return [*torch.autograd.grad(o, leaves, [dh, dy]), *(t.detach() for t in o)]
    first = step()
    assert all(torch.equal(a, c) for a, c in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, held))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", [1, 3, 8, 24, 35, 64, 72, 100, 129, 256])
def test_enough_rows_for_the_ring(C, dtype):
    """Millions of values: the streams through shared memory, samples that end inside a tile, a last
    tile that ends in odd bytes."""
    e = torch.finfo(DT[dtype]).bits // 8
    M = 310 * 12288 // (C * e) + 5
    per = ("gate", "weight", "bias", "next_weight", "next_bias") if C % 3 else ("gate",)
    _run(M, C, 40, DT[dtype], torch.float32, True, "layer", "layer" if C != 1 else "rms", per_sample=per, seed=C)


@pytest.mark.parametrize("norm,next_norm,use", [("none", "none", (True, False)), ("rms", "none", (True, False)),
                                                ("none", "rms", (False, True)), ("rms", "layer", (True, True))])
def test_ring_with_parts_absent(norm, next_norm, use):
    M = 310 * 96 + 7
    _run(M, 64, 3, torch.bfloat16, torch.bfloat16, False, norm, next_norm, residual=False, use=use, seed=11)
    _run(M, 64, 3, torch.bfloat16, torch.bfloat16, True, norm, next_norm, alpha=0.5, use=use, seed=12)


def test_only_the_wanted_gradients():
    x, r, p, off, _, dh, dy = _case(310 * 96, 64, 3, torch.bfloat16, torch.float32, True, "layer", "layer", ("gate",), seed=13)
    named = {"feats": x, "residual": r, **p}

    def grads(wanted):
        full = {k: t.detach().clone().requires_grad_(k in wanted) for k, t in named.items()}
        o = sparse_residual_norm(full["feats"], full["residual"], batch_offsets=off, norm="layer", next_norm="layer",
                                 **{k: full[k] for k in p})
        return torch.autograd.grad(o, [full[k] for k in wanted], [dh, dy])
    every = dict(zip(named, grads(list(named))))
    for k in named:
        assert torch.equal(grads([k])[0], every[k]), k


def test_bad_offsets_of_one_sample_raise():
    x = torch.randn(100, 64, device="cuda")
    gate = torch.randn(1, 64, device="cuda")
    with pytest.raises(RuntimeError, match="sample offsets"):
        sparse_residual_norm(x, x, gate=gate, batch_offsets=torch.tensor([0, 99], dtype=torch.int32, device="cuda"))
        _native.check_errors()
    _native.reset_status()
    hidden, _ = sparse_residual_norm(x, x, gate=gate, batch_offsets=torch.tensor([0, 100], dtype=torch.int32, device="cuda"))
    assert torch.allclose(hidden, x * (1 + gate), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("M,C", [(8_500_001, 256), (1_100_003, 2048)])
def test_more_than_2_to_31_elements(M, C):
    """The first and last rows of a large call equal the same rows alone, forward and backward."""
    x = torch.randn(M, C, device="cuda", dtype=torch.bfloat16)
    for rows in (slice(0, 1000), slice(M - 1000, M)):
        part = x[rows].clone().requires_grad_(True)
        whole = x.detach().requires_grad_(True)
        y, yp = sparse_norm(whole), sparse_norm(part)
        # another lane layout may round a statistic the other way: one rounding of the output
        assert ((y[rows].float() - yp.float()).abs() <= 2.0 ** -7 * yp.float().abs() + 1e-6).all()
        g = torch.autograd.grad(y, whole, x)[0][rows]
        gp = torch.autograd.grad(yp, part, x[rows])[0]
        assert ((g.float() - gp.float()).abs() <= 2.0 ** -7 * gp.float().abs() + 1e-5).all()
        del y, g, whole


def test_second_derivative_is_refused():
    x = torch.randn(10, 8, device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(sparse_norm(x).sum(), x, create_graph=True)
