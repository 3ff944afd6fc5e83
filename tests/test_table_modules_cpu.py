"""CPU tests of the embedding tables: dense gradients from ids outside the table, and the tables as
modules under torch's transforms."""
import pytest
import torch

from collie_amd import functional


@pytest.mark.parametrize('dtype', [torch.int32, torch.int64])
def test_dense_gradient_of_few_rows_takes_no_id_outside_the_table(dtype):
    """(The form of few rows is plain torch, so it can be watched here.)"""
    table = torch.zeros(5, 3)
    bad = [-1, 5, torch.iinfo(dtype).max, torch.iinfo(dtype).min]
    ids = torch.tensor([4, 0, *bad, 0], dtype=dtype)
    vals = torch.arange(1.0, 22.0).reshape(7, 3)
    want = torch.zeros(5, 3)
    want[4], want[0] = vals[0], vals[1] + vals[6]       # whole numbers: exact
    got = functional.table_grad(table, ids, vals)
    assert got.shape == table.shape and got.is_contiguous()
    assert torch.equal(got, want)
    assert torch.equal(functional.table_grad(table, ids[2:6], vals[2:6]), torch.zeros(5, 3))
