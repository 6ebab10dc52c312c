"""The linear layer's gradients that are sums over all rows, where a lost row, tile, split shows.

Integers: sums of small integers are exact in fp32 (here under 2^24), so a gradient equals the exact one
bit for bit, whatever the kernels' order. Few rows with a gradient: the sums then have as many terms, and
the bound is as tight as they are few.
"""
import pytest
import torch

from sparseconv import _native
from sparseconv.ops.linear import sparse_linear

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _ints(gen, *shape, dtype, top=2):
    return torch.randint(-top, top + 1, shape, generator=gen, device="cuda").to(dtype)


def _differs_without(rows, *sums):
    """The exact sums change when the last rows are left out: what a lost tail would give is told apart."""
    assert all((whole != part).any() for whole, part in sums), rows


# CUDA cores (fp32, odd channels), one pass over the rows, separate tensor-core products, pairs of CTAs,
# and copies into whole rows, with ragged last tiles
LINEAR = [(5000, 64, 256), (777, 6, 33), (333, 35, 13), (300000, 32, 13), (1000, 128, 256), (37888, 64, 64),
          (40001, 128, 128), (38000, 8, 8), (41003, 72, 96), (50003, 64, 256), (38001, 24, 136), (200003, 16, 16),
          (300007, 64, 64), (20011, 512, 520), (9473, 520, 1032), (100003, 264, 40), (20001, 257, 131),
          (200001, 129, 72)]


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,Ci,Co", LINEAR)
def test_linear_gradients_of_integers(M, Ci, Co, dtype, act):
    if dtype == "fp32" and M * Ci * Co > 3e9:
        M = int(3e9) // (Ci * Co) + 3
    gen = torch.Generator(device="cuda").manual_seed(M)
    x, g = _ints(gen, M, Ci, dtype=DT[dtype]), _ints(gen, M, Co, dtype=DT[dtype])
    w = _ints(gen, Co, Ci, dtype=torch.float32, top=1).requires_grad_(True)      # fp32: gradients unrounded
    b = _ints(gen, Co, dtype=torch.float32).requires_grad_(True)
    x.requires_grad_(True)
    out = sparse_linear(x, w, b, activation=act)
    gx, gw, gb = torch.autograd.grad(out, [x, w, b], g)
    xd, wd = x.detach().double(), w.detach().double()
    z = xd @ wd.t() + b.detach().double()
    dz = g.double() * (z > 0) if act == "relu" else g.double()
    assert torch.equal(out.detach(), (z.clamp_min(0) if act == "relu" else z).to(DT[dtype]))
    assert torch.equal(gx, (dz @ wd).to(DT[dtype]))
    want_w, want_b = dz.t() @ xd, dz.sum(0)
    assert want_w.abs().max() < 2 ** 24 and torch.equal(gw.double(), want_w) and torch.equal(gb.double(), want_b)
    _differs_without(1, (want_w, dz[:-1].t() @ xd[:-1]) if dz[-1].any() and xd[-1].any() else (1 + want_w, want_w))
    _differs_without(128, (want_w, dz[:-128].t() @ xd[:-128]), (want_b, dz[:-128].sum(0)))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,Ci,Co", [(1, 8, 8), (129, 72, 264), (1000, 512, 520), (4097, 64, 256), (40001, 128, 128),
                                     (20011, 512, 520), (50003, 64, 256)])
def test_tensor_cores_take_these(M, Ci, Co, dtype):
    """With the tensor-core kernels demanded the call is not refused, and gives the bits of the default."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(DT[dtype])
    x, w, b, g = mk(M, Ci), mk(Co, Ci), mk(Co), mk(M, Co)
    runs = []
    for kernel in (_native.KERNEL_AUTO, _native.KERNEL_TCGEN05):
        out, z = _native.linear_forward(x, w, b, None, "gelu", True, kernel)
        runs.append([out, z, *_native.linear_backward(g, z, x, w, "gelu", torch.float32, torch.float32, (True,) * 3, kernel)])
    assert all(torch.equal(a, c) for a, c in zip(*runs))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("M,Ci,Co", [(40001, 128, 128), (50003, 64, 256), (300000, 32, 13), (20011, 512, 520), (20001, 257, 131)])
def test_linear_gradients_of_few_rows(M, Ci, Co, act, dtype):
    """Gradients only in the first and last rows, in the last ragged tile and around tile edges."""
    if dtype == "fp32" and Ci * Co > 1e5:
        M = 3001
    rows = torch.tensor(sorted({0, 1, 127, 128, M // 2, M - 130, M - 128, M - 2, M - 1}), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(M + Ci)
    mk = lambda *s, k=1.0: (torch.randn(*s, generator=gen, device="cuda") * k).to(DT[dtype])
    x, w = mk(M, Ci).requires_grad_(True), mk(Co, Ci, k=Ci ** -0.5).float().requires_grad_(True)
    b = mk(Co).float().requires_grad_(True)
    g = torch.zeros(M, Co, device="cuda", dtype=DT[dtype])
    g[rows] = mk(len(rows), Co)
    gx, gw, gb = torch.autograd.grad(sparse_linear(x, w, b, activation=act), [x, w, b], g)
    xr, gr, wd = x.detach()[rows].double(), g[rows].double(), w.detach().double()
    z = (xr @ wd.t() + b.detach().double()).requires_grad_(True)
    f = {"none": lambda t: t, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[act]
    dz = torch.autograd.grad(f(z), z, gr)[0]
    # dz: the slope's own 2^-20, the product's fp32 steps and its rounding (|act''| <= 0.8), then dz's
    half = torch.finfo(DT[dtype]).eps / 2
    ez = (Ci + 2) * 2.0 ** -23 * (xr.abs() @ wd.abs().t() + b.detach().double().abs())
    e_sum = gr.abs() * (0.0 if act == "none" else 0.8 * (ez + half * (z.detach().abs() + ez) + 2.0 ** -24) + 2.0 ** -20)
    e_dz = e_sum + (0.0 if act == "none" else half * (dz.abs() + e_sum) + 2.0 ** -24)
    n = len(rows)
    steps = (n + 2) * 2.0 ** -23
    for got, want, lim in ((gw, dz.t() @ xr, e_dz.t() @ xr.abs() + steps * ((dz.abs() + e_dz).t() @ xr.abs())),
                           (gb, dz.sum(0), e_sum.sum(0) + steps * (dz.abs() + e_sum).sum(0))):
        lim = lim + 2.0 ** -24 * (want.abs() + lim)
        assert ((got.double() - want).abs() <= lim).all()
        assert (want.abs() > lim).float().mean() > 0.9       # a gradient of zeros is refused
    part = dz[:-1].t() @ xr[:-1]                             # and one without the last row
    lim = e_dz.t() @ xr.abs() + steps * ((dz.abs() + e_dz).t() @ xr.abs())
    assert ((part - dz.t() @ xr).abs() > 2 * lim).float().mean() > 0.5
    lim = e_dz @ wd.abs() + (Co + 2) * 2.0 ** -23 * ((dz.abs() + e_dz) @ wd.abs())
    want = dz @ wd
    assert ((gx[rows].double() - want).abs() <= lim + half * (want.abs() + lim) + 2.0 ** -24).all()
    others = torch.ones(M, dtype=torch.bool, device="cuda")
    others[rows] = False
    assert not gx[others].any()
