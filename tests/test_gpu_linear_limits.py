"""The linear layer's activations where they saturate: kept products beyond the feature dtype's
range, and the far tail of GELU, forward and backward on every path of the kernels.
"""
import pytest
import torch

from sparseconv import _native
from sparseconv.ops.linear import sparse_linear

pytestmark = pytest.mark.gpu

INF = float("inf")


def _slopes(act, dtype, products, M, kernel=_native.KERNEL_AUTO):
    """act'(products[i]), as the gradient of the bias of column i, where the last row's output gradient is one."""
    x = torch.ones(M, 8, device="cuda", dtype=dtype)
    w = torch.zeros(64, 8, device="cuda", dtype=dtype)
    z = torch.zeros(M, 64, device="cuda", dtype=dtype)
    z[:, :len(products)] = torch.tensor(products, device="cuda").to(dtype)
    g = torch.zeros(M, 64, device="cuda", dtype=dtype)
    g[M - 1] = 1.0
    gx, gw, gb = _native.linear_backward(g, z, x, w, act, torch.float32, torch.float32, (True, True, True), kernel)
    # the same slopes, rounded once, times one
    assert torch.allclose(gw, gb[:, None].to(dtype).float().expand(64, 8), rtol=0, atol=0, equal_nan=True)
    assert gx.isnan().all() if products[0] != products[0] else not gx.any()     # W is zero
    return gb[:len(products)].tolist()


# separate kernels on the CUDA cores and the tensor cores, and the one pass over the rows
PATHS = [(5, _native.KERNEL_SIMT), (300, _native.KERNEL_AUTO), (37889, _native.KERNEL_AUTO)]


@pytest.mark.parametrize("M,kernel", PATHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_slopes_at_the_ends(act, dtype, M, kernel):
    """act' is 0 at -inf and 1 at +inf, as everywhere far from 0, and NaN stays NaN."""
    top = torch.finfo(dtype).max
    got = _slopes(act, dtype, [-INF, -top, -200.0, 200.0, top, INF], M, kernel)
    assert [abs(v) for v in got] == [0.0, 0.0, 0.0, 1.0, 1.0, 1.0]
    if act != "relu":
        assert all(v != v for v in _slopes(act, dtype, [float("nan")], M, kernel))


@pytest.mark.parametrize("M", [5, 37889])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_products_beyond_half_precision(act, M):
    """A product of -66,048 in fp16: the output is the activation of it, zero, and so are the gradients
    that pass through it; the rest of the row and of the column is as without it."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(M, 64, generator=g, device="cuda").half()
    w = (torch.randn(64, 64, generator=g, device="cuda") / 8).half()
    w[:, 0] = 0
    w[7, 0] = -258.0
    x[:, 0] = 0
    x[3, 0] = 256.0
    d = torch.randn(M, 64, generator=g, device="cuda").half()
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    out = sparse_linear(x, w, activation=act)
    assert out.isfinite().all() and out[3, 7].abs() < 1e-7
    gx, gw = torch.autograd.grad(out, leaves, d)
    assert gx.isfinite().all() and gw.isfinite().all()
    # the definition: that entry's dz is 0
    z = x.detach().double() @ w.detach().double().t()
    zz = z.clone().requires_grad_(True)
    f = torch.nn.functional
    dz = torch.autograd.grad((f.gelu if act == "gelu" else f.silu)(zz), zz, d.double())[0]
    assert dz[3, 7] == 0
    # dz is off by its rounding, 2^-11, and by the argument's, 2^-11 |z| |act''| (|act''| <= 0.8); twice that
    # covers the fp32 sums; the result by its own rounding
    e = 2 * d.double().abs() * 2.0 ** -11 * (1 + z.abs().clamp_max(20)) + 2.0 ** -24
    for got, want, lim in ((gx, dz @ w.detach().double(), e @ w.detach().double().abs()),
                           (gw, dz.t() @ x.detach().double(), e.t() @ x.detach().double().abs())):
        assert ((got.double() - want).abs() <= lim + 2.0 ** -11 * want.abs() + 2.0 ** -24).all()


def _outputs(act, dtype, z, kernel=_native.KERNEL_AUTO):
    """act at the values of a vector, through a layer that multiplies by one."""
    w = torch.zeros(8, 8, device="cuda", dtype=dtype)
    w[0, 0] = 1.0
    x = torch.zeros(z.numel(), 8, device="cuda", dtype=dtype)
    x[:, 0] = z.to(dtype)
    return x[:, 0].double(), _native.linear_forward(x, w, None, None, act, kernel=kernel)[0][:, 0].double()


def test_negative_tail_in_single_precision():
    """GELU and its slope keep their digits for negative arguments. The argument of the error function is off
    by 2^-23 of itself, its value by z^2 times that, the function by a few steps: (z^2 + 8) 2^-22 in all, for
    the slope (Phi + z phi, which cancel to about -z phi, the second within z^2 2^-23) the same of each term."""
    z0 = torch.linspace(-9.0, 0.0, 5001, device="cuda")
    z, out = _outputs("gelu", torch.float32, z0)
    cdf = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    assert ((out - z * cdf).abs() <= (z * z + 8) * 2.0 ** -22 * (z * cdf).abs()).all()
    x = torch.ones(1, 1, device="cuda")
    w = torch.zeros(z0.numel(), 1, device="cuda")
    d = torch.ones(1, z0.numel(), device="cuda")
    slope = _native.linear_backward(d, z0[None].contiguous(), x, w, "gelu", torch.float32, torch.float32,
                                    (False, False, True))[2].double()
    z, phi = z0.double(), z0.double() * torch.exp(-0.5 * z0.double() ** 2) / (2 * torch.pi) ** 0.5
    cdf = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    assert ((slope - (cdf + phi)).abs() <= (z * z + 8) * 2.0 ** -22 * (cdf + phi.abs())).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_far_tail_in_half_precision(dtype):
    """GELU falls to zero: the fitted tail is within a quarter of the value to -8 and below 1e-17 from there
    on, where Phi is under 7e-16."""
    z, out = _outputs("gelu", dtype, torch.cat([torch.linspace(-9.0, -5.0, 2001, device="cuda"),
                                                torch.tensor([-10.0, -13.0, -14.0, -20.0, -1e3, -6e4], device="cuda")]))
    ref = z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    assert ((out - ref).abs() <= 0.25 * ref.abs() + 1e-17 + (2.0 ** -24 if dtype == torch.float16 else 0.0)).all()
    assert (out[z < -9].abs() <= 1e-17).all() if dtype == torch.bfloat16 else not out[z < -6].any()
