"""What attention and rotary positions refuse, before anything reaches a device."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from sparseconv import _native
from sparseconv.ops.attention import sparse_attention
from sparseconv.ops.rotary import rotary_steps, sparse_rotary

P = 4096


@pytest.fixture(scope="module")
def lib():
    return _native.load_library()


def attention_args(**kw):
    a = _native.AttentionArgs(dtype=1, num_queries=100, num_keys=100, num_samples=2, heads=4, key_heads=2, head_size=64,
                              scale=0.125, offsets=P, key_offsets=P, query=P, key=P, value=P, query_row=256, query_head=64,
                              key_row=128, key_head=64, value_row=128, value_head=64, out=P, row_stats=P, grad_out=P,
                              grad_row=256, grad_head=64, grad_query=P, grad_key=P, grad_value=P, workspace=P, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("field,value,rc", [
    ("dtype", 7, 1), ("kernel", 3, 1), ("num_queries", -1, 1), ("num_queries", 1 << 31, 1), ("num_keys", 1 << 31, 1),
    ("num_samples", 0, 1), ("heads", 3, 1), ("heads", 1, 1), ("key_heads", 0, 1), ("heads", 65538, 1), ("head_size", 0, 1),
    ("head_size", 257, 1), ("scale", 0.0, 1), ("scale", -1.0, 1), ("scale", math.inf, 1), ("scale", math.nan, 1),
    ("offsets", None, 1), ("key_offsets", None, 1), ("query", None, 1), ("key", None, 1), ("value", None, 1), ("out", None, 1),
])
def test_attention_forward(lib, field, value, rc):
    assert lib.spconv_attention_forward(attention_args(**{field: value}), None) == rc
    assert lib.spconv_attention_backward(attention_args(**{field: value}), None) == rc


def test_attention_more(lib):
    fwd, bwd, need = lib.spconv_attention_forward, lib.spconv_attention_backward, lib.spconv_attention_workspace_bytes
    assert fwd(None, None) == 1 and bwd(None, None) == 1 and need(None, 0) == -1
    assert bwd(attention_args(grad_out=None), None) == 1 and bwd(attention_args(row_stats=None), None) == 1
    assert fwd(attention_args(kernel=2, dtype=0), None) == 3 and fwd(attention_args(kernel=2, head_size=136), None) == 3
    assert need(attention_args(), 1) >= 100 * 4 * 4
    assert bwd(attention_args(workspace=None), None) == 1 and bwd(attention_args(workspace=P + 8), None) == 1
    assert bwd(attention_args(workspace_bytes=need(attention_args(), 1) - 1), None) == 1
    assert fwd(attention_args(num_queries=0, query=None, out=None), None) == 0                  # nothing to do
    few = attention_args(num_queries=2, num_keys=100000)
    assert need(few, 0) > 0 and fwd(attention_args(num_queries=2, num_keys=100000, workspace_bytes=need(few, 0) - 1), None) == 1
    for bad in (dict(num_queries=-1), dict(heads=0), dict(head_size=0), dict(num_samples=0), dict(key_heads=3)):
        assert need(attention_args(**bad), 0) == -1
    for nothing in (dict(num_queries=0), dict(num_keys=0), dict(num_queries=0, num_keys=0)):
        for dtype in (0, 1, 2):
            assert need(attention_args(dtype=dtype, **nothing), 0) >= 0 and need(attention_args(dtype=dtype, **nothing), 1) >= 0


@pytest.mark.parametrize("field", ["num_queries", "num_keys"])
def test_rows_whose_tiles_would_pass_32_bits(lib, field):
    """Numbers of a tile's rows and keys are 32-bit, up to a tile past the last row."""
    for rows in ((1 << 31) - 1, (1 << 31) - 1023):
        a = attention_args(**{field: rows})
        assert lib.spconv_attention_forward(a, None) == 1 and lib.spconv_attention_backward(a, None) == 1


def test_attention_python():
    q, k = torch.zeros(10, 4, 64), torch.zeros(12, 2, 64)
    off = torch.tensor([0, 10], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparse_attention(q, q, q)
    with pytest.raises(ValueError, match="batch_offsets"):
        sparse_attention(q, k, k, key_offsets=off)
    with pytest.raises(ValueError, match="as many keys"):
        sparse_attention(q, k, k, off)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sparse_attention(dual, q, q)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sparse_rotary(dual, None, torch.zeros(10, dtype=torch.int32))


@pytest.mark.gpu
def test_attention_shapes_on_the_device():
    q, k = torch.zeros(10, 4, 64, device="cuda"), torch.zeros(10, 2, 64, device="cuda")
    off = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    for args, kind in (((q, k[:, :, :32], k), ValueError), ((q, k, k[:5]), ValueError), ((q[0], k, k), ValueError),
                       ((q, k.half(), k), TypeError), ((q.double(), k.double(), k.double()), TypeError),
                       ((q[:, :3], k, k), ValueError), ((q, k, k, off.long()), ValueError), ((q, k, k, off[:1]), ValueError),
                       ((q, k, k, off, off[:2]), ValueError), ((q, k, k, off.cpu()), RuntimeError)):
        with pytest.raises(kind):
            sparse_attention(*args)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            sparse_attention(q, k, k, scale=scale)
    wide = torch.zeros(2, 1, 257, device="cuda")
    with pytest.raises(ValueError, match="head size"):
        sparse_attention(wide, wide, wide)
    with pytest.raises(NotImplementedError):
        x = q.clone().requires_grad_()
        torch.autograd.grad(sparse_attention(x, k, k).sum(), x, create_graph=True)


def rotary_args(**kw):
    a = _native.RotaryArgs(dtype=1, layout=0, num_rows=10, heads=4, key_heads=2, head_size=64, rotary_dim=64, axes=3, amplitude=1.0,
                           query=P, key=P, query_row=256, query_head=64, key_row=128, key_head=64, query_out=P, key_out=P,
                           positions=P, position_row=3, position_col=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("field,value", [
    ("dtype", 3), ("layout", 2), ("num_rows", -1), ("num_rows", 1 << 31), ("heads", -1), ("heads", 65536), ("head_size", 1),
    ("head_size", 257), ("rotary_dim", 0), ("rotary_dim", 63), ("rotary_dim", 66), ("axes", 0), ("axes", 33), ("query", None),
    ("key_out", None), ("positions", None),
])
def test_rotary(lib, field, value):
    assert lib.spconv_rotary(rotary_args(**{field: value}), None) == 1


def test_rotary_nothing(lib):
    assert lib.spconv_rotary(None, None) == 1 and lib.spconv_rotary(rotary_args(heads=0, key_heads=0), None) == 1
    assert lib.spconv_rotary(rotary_args(num_rows=0, query=None), None) == 0


def test_rotary_python():
    q, pos = torch.zeros(10, 4, 64), torch.zeros(10, 3, dtype=torch.int32)
    for bad in (dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=4), dict(rotary_dim=0), dict(scaling="far"), dict(base=0.0),
                dict(scaling="linear", factor=0.5), dict(factor=2.0), dict(scaling="yarn", factor=2.0), dict(trained_size=5),
                dict(scaling="yarn", factor=2.0, trained_size=0)):
        with pytest.raises(ValueError):
            sparse_rotary(q, None, pos, **bad)
    with pytest.raises(ValueError):
        sparse_rotary(None, None, pos)
    with pytest.raises(ValueError):
        sparse_rotary(q[0], None, pos)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparse_rotary(q, q, pos)


@pytest.mark.gpu
def test_rotary_shapes_on_the_device():
    q, pos = torch.zeros(10, 4, 64, device="cuda"), torch.zeros(10, 3, dtype=torch.int32, device="cuda")
    for args, kind in (((q, q[:5], pos), ValueError), ((q, q.half(), pos), TypeError), ((q, q[:, :, :32], pos), ValueError),
                       ((q, None, pos.long()), TypeError), ((q, None, pos[:5]), ValueError), ((q, None, pos.cpu()), RuntimeError),
                       ((q.double(), None, pos), TypeError), ((torch.zeros(10, 1, 300, device="cuda"), None, pos), ValueError)):
        with pytest.raises(kind):
            sparse_rotary(*args)
    with pytest.raises(ValueError):
        sparse_rotary(q, None, pos, layout="other")


def test_rotary_positions_without_rows():
    with pytest.raises(ValueError, match="positions"):
        sparse_rotary(torch.zeros(10, 4, 64), None, torch.zeros((), dtype=torch.int32))


def test_steps():
    """Scaled steps at both ends of their ranges, by their formulas."""
    plain, one = rotary_steps(16)
    assert one == 1.0 and plain[0] == 1.0 and math.isclose(plain[8], 0.01)
    linear, one = rotary_steps(16, 1e4, "linear", 4.0)
    assert one == 1.0 and all(math.isclose(a, b / 4.0) for a, b in zip(linear, plain))
    ntk, _ = rotary_steps(16, 1e4, "ntk", 4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4.0)
    yarn, amplitude = rotary_steps(16, 1e4, "yarn", 4.0, 1000)
    assert math.isclose(amplitude, 0.1 * math.log(4.0) + 1.0)
    assert yarn[0] == plain[0] and math.isclose(yarn[-1], plain[-1] / 4.0)          # 159 turns, and 0.03
    assert rotary_steps(1, 1e4, "ntk", 4.0)[0] == (1.0,)


def test_turns_are_whole_turns_apart():
    """Steps enter the kernel modulo a turn, in 2^-64ths of it."""
    table = (ctypes.c_uint64 * 128).from_buffer_copy(_native._turn_steps((math.pi, -math.pi / 2, 2.0 * math.pi, 1.0)))
    assert table[0] == 1 << 63 and table[1] == 3 << 62 and table[2] == 0
    assert abs(table[3] / 2.0 ** 64 - 1.0 / (2.0 * math.pi)) < 2.0 ** -53
