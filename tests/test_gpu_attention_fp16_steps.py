"""fp16 training steps, whose samples' largest rows go through the workspace: captured and replayed on other inputs, two graphs and
two streams at once."""
import pytest
import torch

from sparseconv.ops.attention import sparse_attention

pytestmark = pytest.mark.gpu


def step(q, k, v, grad, off, causal):
    out = sparse_attention(q, k, v, off, causal=causal)
    return [out, *torch.autograd.grad(out, (q, k, v), grad)]


def inputs(rows, seed, sizes=(1.0, 1.0)):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, grad = (torch.randn(rows, 2, 64, generator=g, device="cuda") for _ in range(4))
    return [q.half(), k.half(), (v * sizes[0]).half(), (grad * sizes[1]).half()]


@pytest.mark.parametrize("causal", [False, True])
def test_captured_steps(causal):
    off = torch.tensor([0, 300, 300, 420, 1000], dtype=torch.int32, device="cuda")
    buffers = [inputs(1000, 1), inputs(1000, 2)]
    leaves = [[t.clone().requires_grad_() for t in b[:3]] for b in buffers]
    step(*leaves[0], buffers[0][3], off, causal)
    graphs, results = [], []
    for b, leaf in zip(buffers, leaves):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(*leaf, b[3], off, causal))
        graphs.append(graph)
    # gradients and values of other sizes at each replay: what was largest before must not stay
    for sizes in ((1.0, 1.0), (100.0, 2.0 ** 8), (2.0 ** -6, 2.0 ** -10), (1.0, 1.0)):
        fresh = [inputs(1000, 10, sizes), inputs(1000, 11, sizes[::-1] if sizes[0] > 1 else sizes)]
        for new, b, leaf in zip(fresh, buffers, leaves):
            with torch.no_grad():
                for t, n in zip((*leaf, b[3]), new):
                    t.copy_(n)
        for graph in graphs:
            graph.replay()
        for new, got in zip(fresh, results):
            want = step(*(t.clone().requires_grad_() for t in new[:3]), new[3], off, causal)
            assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_streams_at_once():
    off = torch.tensor([0, 700, 3000], dtype=torch.int32, device="cuda")
    sets = [inputs(3000, 3, (1.0, 2.0 ** -10)), inputs(3000, 4, (30.0, 100.0))]
    leaves = [[t.clone().requires_grad_() for t in s[:3]] for s in sets]
    want = [step(*leaf, s[3], off, False) for s, leaf in zip(sets, leaves)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*leaves[i], sets[i][3], off, False))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, w) for run in got[i] for a, w in zip(run, want[i]))
