"""The workspaces that the linear layer's backward asks for stay near what its kernels use."""
import pytest

from sparseconv import _native


def _up(n):
    return (n + 255) // 256 * 256


# the widest 16-bit and fp32 layers of a deep stage, with dz of every row, a split's fp32 weight gradients at
# most a few times over, and the bias sums of 592 row chunks
@pytest.mark.parametrize("dtype,rows,ci,co,most", [
    (2, 20000, 4096, 4096, 1e9), (1, 20000, 1024, 4096, 0.5e9), (2, 20000, 4096, 16384, 2e9), (2, 4000, 16384, 16384, 3e9),
    (2, 84000, 512, 2048, 0.45e9), (0, 20000, 1024, 1024, 0.5e9), (0, 168546, 32, 13, 30e6), (2, 8, 256, 1024, 20e6)])
def test_wide_layers(dtype, rows, ci, co, most):
    f = _native.load_library().spconv_linear_backward_workspace_bytes
    for act in range(4):
        assert 0 < f(dtype, rows, ci, co, act) <= most, (act, f(dtype, rows, ci, co, act))


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("ci,co", [(64, 64), (128, 128), (8, 8), (64, 256), (24, 136), (128, 16)])
@pytest.mark.parametrize("act", [0, 2])
def test_one_pass_shapes(dtype, ci, co, act):
    """Many rows of few channels: the one-pass kernel's sums of each of its 148 CTAs fit as well as the separate
    kernels' (tensors off 16-byte boundaries take those)."""
    f = _native.load_library().spconv_linear_backward_workspace_bytes
    rows = 1_000_000
    one_pass = _up(148 * 8 * co * 4) + _up(148 * co * ci * 4)
    separate = (_up(rows * co * 2) if act else 0) + _up(592 * co * 4)
    if (ci, co, act) != (64, 256, 2):                        # does not fit an SM with its activation
        assert f(dtype, rows, ci, co, act) >= one_pass
    assert f(dtype, rows, ci, co, act) >= separate
