"""Numbers given to rotary positions and attention count by their value at the call: tensors of them too, which may have changed since
the last one, and whose gradients there are not."""
import math
import warnings

import pytest
import torch

from sparseconv.ops.attention import sparse_attention
from sparseconv.ops.rotary import rotary_steps, sparse_rotary


def test_steps_of_a_base_that_changes():
    base, factor = torch.tensor(100.0), torch.tensor(2.0)
    assert rotary_steps(4, base, "linear", factor) == rotary_steps(4, 100.0, "linear", 2.0)
    base.fill_(10000.0)
    factor.fill_(4.0)
    steps, _ = rotary_steps(4, base, "linear", factor)
    assert steps == rotary_steps(4, 10000.0, "linear", 4.0)[0] and all(isinstance(s, float) for s in steps)
    size = torch.tensor(1000)
    first = rotary_steps(4, 1e4, "yarn", 4.0, size)
    size.fill_(50)
    assert first == rotary_steps(4, 1e4, "yarn", 4.0, 1000) and rotary_steps(4, 1e4, "yarn", 4.0, size) == rotary_steps(4, 1e4, "yarn", 4.0, 50)


@pytest.mark.gpu
def test_rotary_by_a_base_that_changes():
    q = torch.randn(5, 2, 16, device="cuda")
    pos = torch.arange(5, device="cuda", dtype=torch.int32)
    base = torch.tensor(100.0)
    assert torch.equal(sparse_rotary(q, None, pos, base=base)[0], sparse_rotary(q, None, pos, base=100.0)[0])
    base.fill_(10000.0)
    assert torch.equal(sparse_rotary(q, None, pos, base=base)[0], sparse_rotary(q, None, pos, base=10000.0)[0])
    scale = torch.tensor(0.5)
    first = sparse_attention(q, q, q, scale=scale)
    scale.fill_(0.25)
    assert torch.equal(first, sparse_attention(q, q, q, scale=0.5)) and torch.equal(sparse_attention(q, q, q, scale=scale), sparse_attention(q, q, q, scale=0.25))


def test_learned_settings_are_refused():
    """Their gradients would be lost without a word. Where none are asked for, they are numbers."""
    q, pos = torch.zeros(10, 4, 64), torch.zeros(10, dtype=torch.int32)
    learned = torch.tensor(2.0, requires_grad=True)
    for call in (lambda: sparse_attention(q, q, q, scale=learned), lambda: sparse_rotary(q, q, pos, base=learned),
                 lambda: sparse_rotary(q, q, pos, scaling="linear", factor=learned),
                 lambda: sparse_rotary(q, q, pos, scaling="yarn", factor=2.0, trained_size=learned)):
        with pytest.raises(NotImplementedError, match="gradient"):
            call()
        with torch.no_grad(), warnings.catch_warnings(), pytest.raises(RuntimeError, match="CUDA"):
            warnings.simplefilter("error")
            call()


@pytest.mark.gpu
def test_scales_past_the_range_are_refused():
    """A score's factor to base 2 is 1.44 times the scale."""
    q = torch.zeros(10, 2, 64, device="cuda")
    for scale in (3e38, 1e39, 1e-50):
        with pytest.raises(ValueError, match="scale"):
            sparse_attention(q, q, q, scale=scale)
    assert math.isfinite(sparse_attention(q, q, q, scale=2.3e38).sum().item())
