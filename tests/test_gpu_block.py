"""A residual block of a sparse network as a user writes it: convolution, norm, feed-forward pair,
gated residual step with the next block's norm, its gradients, and clipping; eager against a
64-bit block of torch operations on the same neighbour map, and captured into a graph.

The fp32 block's sums have at most 27 * 32 products, so a stage's output is off by under 864 half
steps of 2^-24 (5e-5) of its magnitude, about six stages deep each way: 6e-4 of the norm bounds it.
"""
import pytest
import torch

from sparseconv import SparseConvTensor
from sparseconv.ops.clip import clip_gradients
from sparseconv.ops.linear import sparse_linear
from sparseconv.ops.norm import sparse_norm, sparse_residual_norm
from sparseconv.ops.submanifold_conv3d import Algorithm, sparse_submanifold_conv3d

pytestmark = pytest.mark.gpu

C, B = 32, 3


def _setup(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    dense = torch.zeros(B, 12, 12, 12, C)
    occupied = torch.rand(B, 12, 12, 12, generator=g) < 0.3
    dense[occupied] = torch.randn(int(occupied.sum()), C, generator=g)
    x = SparseConvTensor.from_dense(dense.cuda().to(dtype))
    mk = lambda *s, k=1.0, o=0.0: (torch.randn(*s, generator=g) * k + o).cuda().to(dtype).requires_grad_(True)
    p = {"conv": mk(C, 3, 3, 3, C, k=(27 * C) ** -0.5), "conv_b": mk(C, k=0.1), "n1": mk(C, k=0.1, o=1.0), "n1_b": mk(C, k=0.1),
         "up": mk(4 * C, C, k=C ** -0.5), "up_b": mk(4 * C, k=0.1), "down": mk(C, 4 * C, k=(4 * C) ** -0.5),
         "down_b": mk(C, k=0.1), "gate": mk(B, C, k=0.5), "post": mk(C, k=0.1, o=1.0), "next": mk(C, k=0.1, o=1.0)}
    return x, p


def _block(x, feats, p):
    shape = torch.Size((x.batch_size, C, *x.spatial_shape))
    y, cache = sparse_submanifold_conv3d(feats, x.indices, shape, p["conv"], p["conv_b"], None, (1, 1, 1),
                                         Algorithm.IMPLICIT_GEMM)
    y = sparse_norm(y, p["n1"], p["n1_b"])
    y = sparse_linear(y, p["up"], p["up_b"], activation="gelu")
    y = sparse_linear(y, p["down"], p["down_b"], residual=feats)
    hidden, normed = sparse_residual_norm(y, feats, gate=p["gate"], batch_offsets=x.batch_offsets(), residual_scale=0.5,
                                          norm="rms", weight=p["post"], next_norm="rms", next_weight=p["next"])
    return hidden, normed, cache


def _block64(x, feats, p, nbr):
    f = torch.nn.functional
    gathered = torch.where((nbr >= 0)[..., None], feats[nbr.clamp_min(0)], 0.0)
    y = torch.einsum("mvc,ovc->mo", gathered, p["conv"].reshape(C, 27, C)) + p["conv_b"]
    y = f.layer_norm(y, (C,), p["n1"], p["n1_b"], 1e-5)
    y = f.linear(f.gelu(f.linear(y, p["up"], p["up_b"])), p["down"], p["down_b"]) + feats
    rms = lambda t: t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt()
    hidden = 0.5 * feats + p["gate"][x.indices[:, 0].long()] * (rms(y) * p["post"])
    return hidden, rms(hidden) * p["next"]


def _near(got, ref, rel):
    assert (got.double() - ref).norm() <= rel * ref.norm(), ((got.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("dtype,rel", [(torch.float32, 6e-4), (torch.bfloat16, 6e-2)])
def test_block_and_its_gradients(dtype, rel):
    """bf16: about a dozen roundings of 2^-9 on the way to any gradient, 2.4e-2, and each stage's
    gain on those before it of order one: 6e-2."""
    x, p = _setup(dtype)
    feats = x.features.detach().clone().requires_grad_(True)
    hidden, normed, cache = _block(x, feats, p)
    g = torch.Generator(device="cuda").manual_seed(5)
    gh, gn = (torch.randn(hidden.shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    leaves = [feats, *p.values()]
    grads = torch.autograd.grad([hidden, normed], leaves, [gh, gn])
    nbr = cache.neighbor_map.view(torch.int32).long()
    f64 = feats.detach().double().requires_grad_(True)
    p64 = {k: t.detach().double().requires_grad_(True) for k, t in p.items()}
    h64, n64 = _block64(x, f64, p64, nbr)
    ref = torch.autograd.grad([h64, n64], [f64, *p64.values()], [gh.double(), gn.double()])
    _near(hidden.detach(), h64.detach(), rel)
    _near(normed.detach(), n64.detach(), rel)
    for got, want in zip(grads, ref):
        _near(got, want, rel)
    clipped = [torch.empty_like(t) for t in grads]
    total = clip_gradients(grads, 1.0, out=clipped)
    norm64 = sum(t.double().square().sum() for t in grads).sqrt()
    assert abs(total.double() - norm64) < 1e-6 * norm64
    _near(torch.cat([t.flatten() for t in clipped]).float(),
          torch.cat([t.double().flatten() for t in grads]) / (norm64 + 1e-6), 2.0 ** -8)


def test_linear_part_captured():
    """The parts after the convolution, forward and backward and clipping, as one graph."""
    x, p = _setup(torch.bfloat16, seed=1)
    off = x.batch_offsets()
    feats = x.features.detach().clone().requires_grad_(True)
    names = ["up", "up_b", "down", "down_b", "gate", "post", "next"]
    gh = torch.randn_like(feats)

    def step():
        y = sparse_linear(feats, p["up"], p["up_b"], activation="silu")
        y = sparse_linear(y, p["down"], p["down_b"], residual=feats)
        hidden, normed = sparse_residual_norm(y, feats, gate=p["gate"], batch_offsets=off, norm="rms", weight=p["post"],
                                              next_norm="layer", next_weight=p["next"])
        grads = list(torch.autograd.grad([hidden, normed], [feats, *(p[k] for k in names)], [gh, gh]))
        total = clip_gradients(grads, 0.5)
        return [hidden.detach(), normed.detach(), total, *grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        feats.copy_(torch.randn_like(feats))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_refusals_on_device():
    x = torch.randn(8, 16, device="cuda")
    w = torch.randn(24, 16, device="cuda")
    for call, error in (
            (lambda: sparse_linear(x, torch.randn(24, 15, device="cuda")), ValueError),
            (lambda: sparse_linear(x.t(), w), ValueError),
            (lambda: sparse_linear(x[0], w), ValueError),
            (lambda: sparse_linear(x.long(), w), TypeError),
            (lambda: sparse_linear(x, w, torch.randn(23, device="cuda")), ValueError),
            (lambda: sparse_linear(x, w, residual=torch.randn(8, 23, device="cuda")), ValueError),
            (lambda: sparse_linear(x, w, residual=torch.randn(8, 24, device="cuda").half()), TypeError),
            (lambda: sparse_linear(x, w, activation="tanh"), ValueError),
            (lambda: sparse_linear(x, w.cpu()), RuntimeError),
            (lambda: sparse_norm(x, norm="batch"), ValueError),
            (lambda: sparse_norm(x, torch.randn(15, device="cuda")), ValueError),
            (lambda: sparse_norm(x, torch.randn(16, device="cuda").half()), TypeError),
            (lambda: sparse_norm(x, torch.randn(2, 16, device="cuda")), ValueError),
            (lambda: sparse_norm(x, eps=-1.0), ValueError),
            (lambda: sparse_norm(torch.randn(2, 8193, device="cuda")), ValueError),
            (lambda: sparse_norm(x[:, ::2]), ValueError),
            (lambda: sparse_residual_norm(x, x[:4]), ValueError),
            (lambda: sparse_residual_norm(x, x, weight=w[0, :16].contiguous()), ValueError),
            (lambda: sparse_residual_norm(x, x, gate=x, batch_offsets=torch.zeros(9, device="cuda")), ValueError),
            (lambda: sparse_residual_norm(x, x, next_norm="none", next_weight=w[0]), ValueError),
            (lambda: clip_gradients([x.long()], 1.0), TypeError),
            (lambda: clip_gradients([x[:, ::2]], 1.0), ValueError),
            (lambda: clip_gradients([x], 1.0, out=[x[:4]]), ValueError),
            (lambda: clip_gradients([x, x.cpu()], 1.0), RuntimeError)):
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
