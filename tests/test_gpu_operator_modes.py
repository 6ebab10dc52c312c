"""The operators around the convolution in the ways that a training program calls them: saved-tensor
hooks, checkpointing, an input given twice, several streams, and a first call under graph capture."""
import os
import subprocess
import sys
import textwrap

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from sparseconv.ops.clip import clip_gradients
from sparseconv.ops.linear import sparse_linear
from sparseconv.ops.norm import sparse_norm, sparse_residual_norm

pytestmark = pytest.mark.gpu


def _block(x, p, off):
    y = sparse_linear(x, p["up"], p["up_b"], activation="gelu")
    y = sparse_linear(y, p["down"], residual=x)
    return sparse_residual_norm(y, x, gate=p["gate"], batch_offsets=off, norm="layer", weight=p["w"], next_norm="rms")


def _setup(M, C=64, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s, k=1.0, t=dtype: (torch.randn(*s, generator=g, device="cuda") * k).to(t).requires_grad_(True)
    x = mk(M, C)
    p = {"up": mk(2 * C, C, k=C ** -0.5), "up_b": mk(2 * C), "down": mk(C, 2 * C, k=(2 * C) ** -0.5),
         "gate": mk(2, C, t=torch.float32), "w": mk(C, t=torch.float32)}
    return x, p, torch.tensor([0, M // 3, M], dtype=torch.int32, device="cuda"), torch.randn_like(x)


def _grads(outs, x, p, d):
    return torch.autograd.grad(list(outs), [x, *p.values()], [d, d])


@pytest.mark.parametrize("M", [300, 40000])
def test_saved_on_the_host_and_checkpointed(M):
    x, p, off, d = _setup(M)
    want = _grads(_block(x, p, off), x, p, d)
    with torch.autograd.graph.save_on_cpu():
        outs = _block(x, p, off)
    churn = [torch.full_like(x, 7.0) for _ in range(4)]       # what the forward's tensors left is written over
    got = _grads(outs, x, p, d)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del churn
    for reentrant in (False, True):
        outs = checkpoint(_block, x, p, off, use_reentrant=reentrant)
        for t in (x, *p.values()):
            t.grad = None
        torch.autograd.backward(list(outs), [d, d])
        if reentrant:                        # parameters inside a dictionary get theirs as leaves
            assert torch.equal(x.grad, want[0])
        assert all(torch.equal(t.grad, c) for t, c in zip((x, *p.values()), want))


@pytest.mark.parametrize("M", [300, 40000])
def test_one_tensor_as_two_inputs(M):
    """The features as their own residual: the gradients add."""
    x, p, off, d = _setup(M)
    w = p["up"].detach()[:64].contiguous()
    twin = x.detach().clone().requires_grad_(True)
    for f in (lambda a, b: sparse_linear(a, w, residual=b, activation="silu"), lambda a, b: sparse_norm(a) + 0 * b,
              lambda a, b: sparse_residual_norm(a, b, norm="layer", next_norm="none")[0]):
        one = f(x, x)
        two = f(x, twin)
        assert torch.equal(one, two)
        ga, gb = torch.autograd.grad(two, [x, twin], d)
        assert torch.equal(torch.autograd.grad(one, x, d)[0], ga + gb)


def test_streams_at_once():
    cases = [_setup(60000, seed=s) for s in (1, 2)]

    def step(x, p, off, d):
        outs = _block(x, p, off)
        grads = _grads(outs, x, p, d)
        clipped = [torch.empty_like(t) for t in grads]
        return [*(t.detach() for t in outs), clip_gradients(grads, 0.5, out=clipped), *clipped]
    want = [step(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(step(*c))
    torch.cuda.synchronize()
    for runs, ref in zip(got, want):
        for run in runs:
            assert all(torch.equal(a, c) for a, c in zip(run, ref))


def test_backward_of_a_thread_whose_first_call_is_captured():
    """A forward outside, then a capture that holds the process's first backward of the linear layer."""
    code = textwrap.dedent("""
        import torch
        from sparseconv.ops.linear import sparse_linear
        x = torch.randn(40000, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.randn(64, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        d = torch.randn_like(x)
        with torch.no_grad():
            sparse_linear(x, w)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = torch.autograd.grad(sparse_linear(x, w, activation="relu"), [x, w], d)
        graph.replay()
        torch.cuda.synchronize()
        ref = torch.autograd.grad(sparse_linear(x, w, activation="relu"), [x, w], d)
        assert all(torch.equal(a, b) for a, b in zip(held, ref))
        print("captured")
    """)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "sparse-conv_b200"), SPARSECONV_SYNC_CHECK="0")
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
