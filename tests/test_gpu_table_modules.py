"""
GPU tests (``-m gpu``) of embedding lookups at the edges of what a caller may do with them: ids outside
the table, and the tables called as modules under torch's transforms.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')


@pytest.mark.parametrize('padding', [None, 2])
@pytest.mark.parametrize('bad', ['some', 'all'])
def test_sparse_gradient_leaves_out_ids_outside_the_table(bad, padding):
    from collie_amd import functional as F
    w = torch.randn(6, 4, generator=torch.Generator().manual_seed(0)).to(DEV).requires_grad_()
    ids = torch.tensor([[5, 6, -1], [1, 1 << 40, 1], [2, -(1 << 40), 0]] if bad == 'some'
                       else [[6, -1, 7]], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = F.embedding_rows(w, ids, scale=0.5, sparse=True, padding_idx=padding, status=status)
    (g,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert g.is_sparse and g.shape == (6, 4) and status.item() == 1
    rows = g._indices()[0].cpu().tolist()
    want = [r for r in ids.reshape(-1).tolist() if 0 <= r < 6 and r != padding]
    assert rows == want and g._values().shape == (len(want), 4)
    assert (g._values() == 0.5).all()       # exact: one factor of one half
