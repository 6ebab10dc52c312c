"""The CUDA-core attention kernels of 16-bit tensors at the head sizes that the tensor cores take when left to choose: against
64 bits."""
import math

import pytest
import torch

from sparseconv import _native

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def ends(lengths):
    return torch.tensor([0, *lengths], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def reference(q, k, v, lengths, key_lengths, causal, grad):
    G = q.shape[1] // k.shape[1]
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    outs, i0, j0 = [], 0, 0
    for n, m in zip(lengths, key_lengths):
        a = leaves[0][i0:i0 + n]
        b, c = (t[j0:j0 + m].repeat_interleave(G, 1) for t in leaves[1:])
        s = torch.einsum("ihd,jhd->hij", a, b) * q.shape[2] ** -0.5
        hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1) & causal
        p = s.masked_fill(hidden, -math.inf).softmax(-1).masked_fill(hidden.all(1)[:, None], 0.0) if m else s
        outs.append(torch.einsum("hij,jhd->ihd", p, c))
        i0, j0 = i0 + n, j0 + m
    out = torch.cat(outs)
    return [out.detach(), *torch.autograd.grad(out, leaves, grad.double())]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 8, 31, 32, 33, 48, 64, 72, 96, 127, 128])
@pytest.mark.parametrize("lengths,key_lengths,H,K,causal", [
    ([70, 129, 30], [70, 129, 30], 2, 2, False),
    ([70, 0, 129], [40, 9, 200], 4, 2, True),
    ([200], [130], 3, 1, True),
    ([1, 2], [3000, 4500], 8, 1, False),         # splits
    ([2500], [5], 2, 2, False),                  # splits of the queries, for the keys' gradients
])
def test_against_64_bits(dtype, D, lengths, key_lengths, H, K, causal):
    """Products and sums are fp32, so that out's, the kept rest's and the gradients' own rounding is all: half a step each, and
    none enters another but out's in delta, with the rest beside it."""
    g = torch.Generator(device="cuda").manual_seed(D)
    M, N = sum(lengths), sum(key_lengths)
    q, k, v, grad = (torch.randn(r, h, D, generator=g, device="cuda").to(dtype) for r, h in ((M, H), (N, K), (N, K), (M, H)))
    off, key_off = ends(lengths), ends(key_lengths)
    out, stats, args = _native.attention_forward(q, k, v, off, key_off, causal, D ** -0.5, keep_stats=True, kernel=_native.KERNEL_SIMT)
    assert args.kernel == _native.KERNEL_SIMT
    grads = _native.attention_backward_of(args, q, k, v, off, key_off, out, stats, grad, (True, True, True))
    for name, got, want in zip("oqkv", (out, *grads), reference(q, k, v, lengths, key_lengths, causal, grad)):
        assert got.dtype == dtype
        norm = want.norm().item()
        assert ((got.double() - want).norm().item() <= torch.finfo(dtype).eps / 2 * norm), (name, (got.double() - want).norm().item() / norm)
