"""``SparseConvTensor.batch_offsets``: first rows of the samples, or offsets that every use refuses where
the rows are not in batch order."""
import pytest
import torch

from sparseconv import SparseConvTensor, _native
from sparseconv.ops.norm import sparse_residual_norm


def _tensor(column, batch, device="cpu", dtype=torch.int32):
    ind = torch.zeros(len(column), 4, dtype=dtype, device=device)
    ind[:, 0] = torch.tensor(column, dtype=dtype, device=device)
    return SparseConvTensor(torch.randn(len(column), 16, device=device), ind, [4, 4, 4], batch)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("column,batch,want", [([0, 0, 2, 2, 2], 4, [0, 2, 2, 5, 5]), ([], 2, [0, 0, 0]), ([0], 1, [0, 1]),
                                               ([1, 1], 2, [0, 0, 2]), ([0] * 7, 1, [0, 7])])
def test_rows_in_batch_order(column, batch, want, dtype):
    off = _tensor(column, batch, dtype=dtype).batch_offsets()
    assert off.tolist() == want and off.dtype == torch.int32


@pytest.mark.parametrize("column,batch", [([1, 0], 2), ([0, 2, 1, 2], 3), ([0, 1, 0, 1, 1], 2), ([2, 2, 2, 0], 3)])
def test_other_rows_give_offsets_that_no_call_takes(column, batch):
    """A binary search over such a column can still ascend from 0 to the number of rows."""
    off = _tensor(column, batch).batch_offsets()
    assert off.tolist() == [-1] * (batch + 1) and off.dtype == torch.int32


def test_batch_numbers_outside_the_batch():
    for column in ([-1, 0, 1], [0, 1, 2]):
        off = _tensor(column, 2).batch_offsets().tolist()
        assert off[0] != 0 or off[-1] != 3


@pytest.mark.gpu
def test_residual_step_refuses_unordered_rows():
    t = _tensor([0, 1, 0, 1, 1], 2, "cuda")
    gate = torch.randn(2, 16, device="cuda")
    with pytest.raises(RuntimeError, match="sample offsets"):
        sparse_residual_norm(t.features, t.features, gate=gate, batch_offsets=t.batch_offsets())
        _native.check_errors()
    _native.reset_status()
    order = t.indices[:, 0].sort(stable=True).indices
    t = SparseConvTensor(t.features[order], t.indices[order], [4, 4, 4], 2)
    hidden, _ = sparse_residual_norm(t.features, t.features, gate=gate, batch_offsets=t.batch_offsets(), next_norm="none")
    _native.check_errors()
    assert torch.allclose(hidden, t.features * (1 + gate[[0, 0, 1, 1, 1]]), rtol=1e-6, atol=1e-6)
