"""The bounded waits of the linear and norm kernels, exercised on the GPU without a fault: with the
limit at 1 ns the first wait that is not already satisfied gives up, the kernel waits (bounded) for
its own copies and MMAs and returns, the host sees the status as a ``RuntimeError``, and with the
default limit the same call on the same context gives the result it gave before."""
import pytest
import torch

from sparseconv import _native

pytestmark = pytest.mark.gpu


def _linear(M, Ci, Co, act="gelu"):
    g = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    x, w, b, r = mk(M, Ci), mk(Co, Ci), mk(Co), mk(M, Co)
    return lambda: list(_native.linear_forward(x, w, b, r, act, keep_preact=True))


def _linear_backward(M, Ci, Co):
    g = torch.Generator(device="cuda").manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    x, w, z, d = mk(M, Ci), mk(Co, Ci), mk(M, Co), mk(M, Co)
    return lambda: list(_native.linear_backward(d, z, x, w, "gelu", torch.bfloat16, torch.bfloat16, (True, True, True)))


def _norm(M, C, backward):
    g = torch.Generator(device="cuda").manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, r, d = (mk(M, C).to(torch.bfloat16) for _ in range(3))
    ps = (mk(2, C), mk(C), mk(C), mk(C), mk(C))
    off = torch.tensor([0, M // 3, M], dtype=torch.int32, device="cuda")
    fwd = lambda: list(_native.residual_norm_forward(x, r, ps, off, 1.0, "layer", "layer", 1e-5, keep_stats=True)[:3])
    if not backward:
        return fwd
    stats = fwd()[2]
    return lambda: _native.residual_norm_backward(x, r, ps, off, 1.0, "layer", "layer", 1e-5, stats, d, d, (True,) * 7)


@pytest.mark.parametrize("make", [
    lambda: _linear(5000, 64, 64), lambda: _linear(50000, 64, 256), lambda: _linear(3000, 1024, 256),
    lambda: _linear(20000, 512, 520), lambda: _linear_backward(40000, 128, 128), lambda: _linear_backward(20000, 512, 520),
    lambda: _norm(60000, 64, False), lambda: _norm(60000, 64, True)],
    ids=["linear", "linear_resident", "linear_streamed", "linear_pairs", "backward_one_pass", "backward_pairs", "norm",
         "norm_backward"])
def test_wait_timeout_is_reported_and_the_context_stays_usable(make):
    call = make()
    ref = call()
    torch.cuda.synchronize()
    prev = _native.set_wait_limit_ns(1)
    try:
        with pytest.raises(RuntimeError, match="wait reached its time limit"):
            call()
            _native.check_errors()
    finally:
        _native.set_wait_limit_ns(prev)
    torch.cuda.synchronize()
    _native.reset_status()
    again = call()
    torch.cuda.synchronize()
    assert _native.check_errors() == 0
    assert all(torch.equal(a, b) for a, b in zip(again, ref))
