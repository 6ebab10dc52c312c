"""A problem that a kernel reported in the host's status word is raised by the next call that checks,
of whatever kind, not only by those whose kernels write there."""
import ctypes

import pytest
import torch

from sparseconv import SparseConvTensor, _native
from sparseconv.ops.clip import clip_gradients
from sparseconv.ops.linear import sparse_linear
from sparseconv.ops.norm import sparse_norm
from sparseconv.ops.submanifold_conv3d import Algorithm, sparse_submanifold_conv3d


class _Status:
    def __init__(self, bits):
        self.pending = False
        self.mapped_word = ctypes.c_int32(bits)
        self.mapped_ptr = ctypes.addressof(self.mapped_word)


@pytest.mark.parametrize("bits,text", [(_native.STATUS_WAIT_TIMEOUT, "time limit"), (_native.STATUS_OFFSETS, "sample offsets")])
@pytest.mark.parametrize("check", [lambda: _native.before_launch(torch.device("cuda", 0)), lambda: _native.mapped_status(0)],
                         ids=["before_launch", "mapped_status"])
def test_both_checks_read_it(monkeypatch, check, bits, text):
    monkeypatch.setattr(_native, "_status", {0: _Status(bits)})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with pytest.raises(RuntimeError, match=text):
        check()
    check()                                  # reported once


def test_not_while_a_stream_is_captured(monkeypatch):
    """The convolution's checks wait for the end of a capture."""
    st = _Status(_native.STATUS_OFFSETS)
    monkeypatch.setattr(_native, "_status", {0: st})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    _native.before_launch(torch.device("cuda", 0))
    assert st.mapped_word.value == _native.STATUS_OFFSETS


@pytest.mark.gpu
def test_every_kind_of_call_raises():
    x = SparseConvTensor.from_dense(torch.ones(1, 4, 4, 4, 16, device="cuda", dtype=torch.float16))
    shape, w = torch.Size((1, 16, 4, 4, 4)), torch.randn(16, 3, 3, 3, 16, device="cuda", dtype=torch.float16) * 0.05
    f = x.features
    leaf = f.clone().requires_grad_(True)

    def conv(feats=f, cache=None):
        return sparse_submanifold_conv3d(feats, x.indices, shape, w, None, cache, (1, 1, 1), Algorithm.IMPLICIT_GEMM)
    _, cache = conv()
    out, _ = conv(leaf, cache)
    st = _native.status_word(f.device)
    calls = {"map and convolution": conv, "convolution": lambda: conv(f, cache), "dense": x.dense,
             "backward": lambda: torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True),
             "linear": lambda: sparse_linear(f, w[:, 0, 0, 0]), "norm": lambda: sparse_norm(f),
             "clipping": lambda: clip_gradients([f.clone()], 1.0)}
    for name, call in calls.items():
        call()
        st.mapped_word.value = _native.STATUS_OFFSETS
        with pytest.raises(RuntimeError, match="sample offsets"):
            call()
            pytest.fail(name)
        assert st.mapped_word.value == 0
        call()
    _native.check_errors()
