"""What the linear, norm and clipping entry points refuse, before anything reaches a device."""
import ctypes

import pytest
import torch

from sparseconv import _native
from sparseconv.ops.clip import clip_grad_norm_, clip_gradients
from sparseconv.ops.linear import sparse_linear
from sparseconv.ops.norm import sparse_norm, sparse_residual_norm

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    return _native.load_library()


def test_linear_forward(lib):
    f = lib.spconv_linear_forward
    assert f(P, 7, 10, 8, P, None, None, 8, 0, P, None, None, 0, 0, None, None) == 1            # dtype
    assert f(P, 0, -1, 8, P, None, None, 8, 0, P, None, None, 0, 0, None, None) == 1            # rows
    assert f(P, 0, 1 << 31, 8, P, None, None, 8, 0, P, None, None, 0, 0, None, None) == 1
    assert f(P, 0, 10, 0, P, None, None, 8, 0, P, None, None, 0, 0, None, None) == 1            # channels
    assert b"channels" in lib.spconv_last_error()
    assert f(P, 0, 10, 8, P, None, None, 65537, 0, P, None, None, 0, 0, None, None) == 1
    assert f(P, 0, 10, 8, P, None, None, 8, 4, P, None, None, 0, 0, None, None) == 1            # activation
    assert f(P, 0, 10, 8, P, None, None, 8, 0, P, None, None, 0, 3, None, None) == 1            # kernel choice
    assert f(None, 0, 10, 8, P, None, None, 8, 0, P, None, None, 0, 0, None, None) == 1         # null
    assert f(P, 0, 10, 8, P, None, None, 8, 0, P, None, None, 0, 2, None, None) == 3            # tcgen05: no fp32
    assert f(None, 0, 0, 8, None, None, None, 8, 0, None, None, None, 0, 0, None, None) == 0    # no rows
    need = lib.spconv_linear_forward_workspace_bytes(2, 50000, 257, 131, 1, 0)
    assert need > 50000 * (264 + 2 * 136) * 2 and lib.spconv_linear_forward_workspace_bytes(2, 50000, 256, 128, 1, 1) == 0
    for m, ci, co in ((20000, 257, 131), (15000, 1001, 517), (200001, 129, 72)):            # shapes that are copied
        assert lib.spconv_linear_forward_workspace_bytes(1, m, ci, co, 0, 0) > 0
    assert lib.spconv_linear_forward_workspace_bytes(0, 50000, 257, 131, 1, 0) == 0          # fp32: no tensor cores
    assert lib.spconv_linear_forward_workspace_bytes(2, 50000, 0, 131, 1, 0) == -1
    assert f(P, 2, 50000, 257, P, None, P, 131, 0, P, None, P, need - 1, 0, None, None) == 1
    assert f(P, 2, 50000, 257, P, None, P, 131, 0, P, None, ctypes.c_void_p(8), need, 0, None, None) == 1


def test_linear_backward(lib):
    f, ws = lib.spconv_linear_backward, lib.spconv_linear_backward_workspace_bytes
    need = ws(1, 100, 16, 24, 2)
    assert need >= 100 * 24 * 2 and ws(9, 1, 1, 1, 0) == -1 and ws(0, 1, 0, 1, 0) == -1
    ok = [P, P, P, P, 1, 100, 16, 24, 2, P, P, 0, P, 1, P, need, 0, None, None]

    def refused(at, value, rc=1):
        args = list(ok)
        args[at] = value
        return f(*args) == rc
    assert refused(0, None) and refused(1, None) and refused(2, None) and refused(3, None)
    assert refused(11, 2) and refused(13, 2)                 # gradient types: fp32 or the features'
    assert refused(14, None) and refused(15, need - 1) and refused(14, ctypes.c_void_p(8))
    assert refused(8, -1)


def test_residual_norm(lib):
    fwd, bwd = lib.spconv_residual_norm_forward, lib.spconv_residual_norm_backward
    A = _native.ResidualNormArgs
    base = dict(dtype=0, channels=16, num_rows=10, feats=256, hidden=256, normed=256, num_samples=1, norm=1,
                next_norm=2, residual_scale=1.0, eps=1e-5)

    def rc(fn, **kw):
        return fn(A(**{**base, **kw}), None)
    assert fwd(None, None) == 1
    for kw in (dict(dtype=5), dict(num_rows=-1), dict(num_rows=1 << 31), dict(channels=0), dict(channels=8193),
               dict(norm=3), dict(next_norm=-1), dict(num_samples=0), dict(num_samples=65536), dict(feats=None),
               dict(hidden=None), dict(normed=None)):
        assert rc(fwd, **kw) == 1, kw
    per = _native.ChannelParam(data=256, dtype=0, per_sample=1)
    assert rc(fwd, gate=per, num_samples=3) == 1 and b"offsets" in lib.spconv_last_error()
    assert rc(fwd, gate=_native.ChannelParam(data=256, dtype=2)) == 1      # bf16 gate, fp32 features
    assert rc(fwd, gate=_native.ChannelParam(grad=256)) == 1
    assert rc(bwd) == 1 and b"gradient" in lib.spconv_last_error()
    assert rc(bwd, grad_hidden=256, gate=_native.ChannelParam(data=256, grad=256)) == 1   # no workspace
    assert b"workspace" in lib.spconv_last_error()
    assert lib.spconv_residual_norm_workspace_bytes(10, 16, 3) > 0
    assert lib.spconv_residual_norm_workspace_bytes(10, 8193, 1) == -1
    assert rc(fwd, num_rows=0, feats=None) == 0


def test_clip_gradients(lib):
    f, need = lib.spconv_clip_gradients, lib.spconv_clip_gradients_workspace_bytes(2)

    def call(ptrs, outs, sizes, codes, n=None, kind=0, limit=1.0, total=256, ws=256, nbytes=need):
        n = len(ptrs) if n is None else n
        U, I, C = ctypes.c_void_p * len(ptrs), ctypes.c_int64 * len(ptrs), ctypes.c_int32 * len(ptrs)
        return f(U(*ptrs), U(*outs), I(*sizes), C(*codes), n, kind, limit, total, ws, nbytes, None)
    assert call([256], [256], [4], [0], n=-1) == 1
    assert call([256], [256], [4], [0], kind=2) == 1
    assert call([256], [256], [4], [0], limit=-1.0) == 1 and call([256], [256], [4], [0], limit=float("nan")) == 1
    assert call([256], [256], [4], [0], total=None) == 1
    assert call([256], [256], [4], [9]) == 1 and call([256], [256], [-4], [0]) == 1
    assert call([None], [256], [4], [0]) == 1 and call([256], [None], [4], [0]) == 1
    assert call([256], [256], [4], [0], ws=None) == 1 and call([256], [256], [4], [0], nbytes=8) == 1
    assert f(None, None, None, None, 1, 0, 1.0, 256, 256, need, None) == 1
    # overlaps: the same tensor twice, outputs into other gradients, a gradient reaching into an output
    assert call([256, 256], [256, 256], [4, 4], [0, 0]) == 1 and b"overlap" in lib.spconv_last_error()
    assert call([256, 264], [256, 264], [4, 4], [0, 0]) == 1
    assert call([256, 512], [512, 256], [4, 4], [0, 0]) == 1
    assert call([256, 512], [1024, 260], [100, 4], [0, 0]) == 1
    assert call([256, 300], [1024, 300], [100, 4], [0, 0]) == 1
    assert call([256], [258], [4], [1]) == 1
    assert lib.spconv_clip_gradients_workspace_bytes(-1) == -1


def test_cpu_tensors_raise():
    x, w = torch.randn(4, 8), torch.randn(8, 8)
    for call in (lambda: sparse_linear(x, w), lambda: sparse_norm(x), lambda: clip_gradients([x], 1.0),
                 lambda: sparse_residual_norm(x, x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_clip_arguments():
    x = torch.randn(4)
    with pytest.raises(ValueError):
        clip_gradients([], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([x], -1.0)
    with pytest.raises(ValueError):
        clip_gradients([x], float("nan"))
    with pytest.raises(ValueError):
        clip_gradients([x], 1.0, norm_type=1.0)
    with pytest.raises(ValueError):
        clip_gradients([x], 1.0, out=[x, x])
    p = torch.nn.Parameter(x)
    assert clip_grad_norm_([p], 1.0).item() == 0.0
