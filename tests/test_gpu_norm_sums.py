"""The residual norm's gradients that are sums over all rows, where a lost row, tile, record shows.

Integers: sums of small integers are exact in fp32 (here under 2^24), so a gradient equals the exact one
bit for bit, whatever the kernels' order. Few rows with a gradient: the sums then have as many terms, and
the bound is as tight as they are few.
"""
import pytest
import torch

from sparseconv.ops.norm import sparse_residual_norm
from test_gpu_norm import U, _case, _ref

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _ints(gen, *shape, dtype, top=2):
    return torch.randint(-top, top + 1, shape, generator=gen, device="cuda").to(dtype)


def _rows_of(C, dtype):
    """Rows enough for the streams through shared memory."""
    return 310 * 12288 // (C * torch.finfo(DT[dtype]).bits // 8) + 5


def _samples(M, B, seed):
    """Row offsets of B samples, some of them empty, and each row's sample."""
    gen = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, M + 1, (B - 1,), generator=gen).sort().values
    cuts[0], cuts[B // 2] = 0, cuts[B // 2 - 1]
    off = torch.cat([torch.tensor([0]), cuts, torch.tensor([M])]).to(torch.int32).cuda()
    return off, torch.repeat_interleave(torch.arange(B, device="cuda"), (off[1:] - off[:-1]).long())


SHAPES = [("ring", C) for C in (1, 3, 8, 24, 32, 35, 64, 72, 100, 129, 256)] + \
         [(M, C) for M, C in ((1, 64), (700, 35), (5000, 64), (20011, 128), (4001, 300), (9001, 520), (3000, 1032), (2003, 2050),
                              (1500, 8192))]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,C", SHAPES)
def test_norm_sums_of_integers(M, C, dtype):
    """The gate's gradient without norms (sums of dh * x), and those of both biases (sums of dh and of dy,
    without a gate), per sample, of integers: exact."""
    M = _rows_of(C, dtype) if M == "ring" else M
    B = 37
    off, sample = _samples(M, B, C)
    gen = torch.Generator(device="cuda").manual_seed(C)
    x, r, dh, dy = (_ints(gen, M, C, dtype=DT[dtype]) for _ in range(4))

    def sums(v):
        return torch.zeros(B, C, dtype=torch.float64, device="cuda").index_add_(0, sample, v)
    gate = torch.ones(B, C, device="cuda", requires_grad=True)
    hidden, _ = sparse_residual_norm(x, r, gate=gate, batch_offsets=off, next_norm="none")
    assert torch.equal(hidden.detach(), x + r)
    want = sums(dh.double() * x.double())
    assert torch.equal(torch.autograd.grad(hidden, gate, dh)[0].double(), want)
    w, b, nb = torch.ones(C, device="cuda"), *(torch.zeros(B, C, device="cuda", requires_grad=True) for _ in range(2))
    hidden, normed = sparse_residual_norm(x, r, batch_offsets=off, norm="layer", weight=w, bias=b, next_norm="rms",
                                          next_bias=nb)
    assert torch.equal(torch.autograd.grad(normed, nb, dy, retain_graph=True)[0].double(), sums(dy.double()))
    assert torch.equal(torch.autograd.grad(hidden, b, dh)[0].double(), sums(dh.double()))
    # one row for all samples
    nb1, b1 = (torch.zeros(C, device="cuda", requires_grad=True) for _ in range(2))
    hidden, normed = sparse_residual_norm(x, r, gate=gate.detach(), batch_offsets=off, norm="layer", weight=w, bias=b1,
                                          next_norm="rms", next_bias=nb1)
    assert torch.equal(torch.autograd.grad(normed, nb1, dy, retain_graph=True)[0].double(), dy.double().sum(0))
    assert torch.equal(torch.autograd.grad(hidden, b1, dh)[0].double(), dh.double().sum(0))
    if M > 128:
        tail = dh[-128:].double().sum(0)
        assert tail.any() and (dh[-128:].double() * x[-128:].double()).sum(0).any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,C", [(m, c) for m, c in SHAPES if c > 1 and (m == "ring" or m > 64)])
def test_norm_sums_of_few_rows(M, C, dtype):
    """All five parameters' gradients where only few rows have one: the first and last, rows on either side
    of every sample's border and of tiles' edges."""
    M = _rows_of(C, dtype) if M == "ring" else M
    B = 9
    per = ("gate", "weight", "bias", "next_weight", "next_bias")
    x, r, p, _, _, dh, dy = _case(M, C, B, DT[dtype], torch.float32, True, "layer", "layer", per, seed=C)
    off, sample = _samples(M, B, C + 1)
    edges = [o + d for o in off.tolist() for d in (-1, 0)] + [0, 1, 7, 8, 255, 256, M // 2, M - 2, M - 1]
    rows = torch.tensor(sorted({e for e in edges if 0 <= e < M}), device="cuda")
    for d in (dh, dy):
        keep = d[rows]
        d.zero_()
        d[rows] = keep
    leaves = [t.requires_grad_(True) for t in (x, r, *p.values())]
    out = sparse_residual_norm(x, r, batch_offsets=off, norm="layer", next_norm="layer", **p)
    grads = torch.autograd.grad(out, leaves, [dh, dy])
    ref = _ref(x.detach()[rows], r.detach()[rows], *(t.detach() for t in p.values()), sample[rows], 1.0, "layer", "layer",
               dh[rows], dy[rows])
    told = []
    for name, got in zip(("feats", "residual", *p), grads):
        want, bound = ref[name]
        if name in ("feats", "residual"):
            assert not got[[i for i in (2, 3, M - 3) if i not in rows]].any()
            got = got[rows]
        lim = bound + torch.finfo(got.dtype).eps / 2 * (want.abs() + bound) + 2.0 ** -24 * (got.dtype == torch.float16) + 1e-37
        assert ((got.double() - want).abs() <= lim).all(), name
        if name not in ("feats", "residual"):
            has = torch.zeros(B, dtype=torch.bool, device="cuda").index_fill(0, sample[rows], True)
            told.append((want.abs() > 2 * lim)[has].float().mean().item())
            assert not got[~has].any()
    assert min(told) > 0.8, told                             # gradients of zeros are refused


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", [64, 128, 256])
@pytest.mark.parametrize("M", [500, 310 * 96])
def test_first_channels_unlike_the_rest(M, C, dtype):
    """LayerNorm of rows whose first eight values are a thousand times the others.

    fp32 takes the mean first and squares the deviations: a mean of squares passes at most 22 roundings of U, so
    1 / deviation is off by 11 U and a few steps, and the values by their mean's and their own, 18 U of the
    largest; where the squares are taken around a shift s, var = mean(d^2) - mean(d)^2, and (s - mean)^2 is at
    most C / 8 - 1 variances where s is the mean of eight of the row's values: both terms are under C / 8
    variances, and with 14 roundings in the first, 20 in the second and 2 more (C / 8 + 1) 36 U of the variance
    are lost, half of it of 1 / deviation. That is for 16-bit features, whose own rounding is far above it.
    """
    gen = torch.Generator(device="cuda").manual_seed(C)
    x = torch.randn(M, C, generator=gen, device="cuda")
    x[:, :8] = x[:, :8] * 10 + 1000.0
    x = x.to(DT[dtype])
    hidden, _ = sparse_residual_norm(x, norm="layer", next_norm="none", eps=1e-5)
    xd = x.double()
    d = xd - xd.mean(1, keepdim=True)
    rstd = (d.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    want = d * rstd
    lim = (15 if dtype == "fp32" else (C / 8 + 1) * 18 + 4) * U * want.abs() + 18 * U * xd.abs().amax(1, keepdim=True) * rstd
    assert ((hidden.double() - want).abs() <= lim + torch.finfo(DT[dtype]).eps / 2 * (want.abs() + lim)).all()
