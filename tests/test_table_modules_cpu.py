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


# ---- the tables as modules under torch's transforms ------------------------------------------------
IDS = torch.tensor([0, 4, 4, 1])


def _table():
    from collie_amd import layers
    torch.manual_seed(0)
    return layers.ScaledEmbedding(5, 3)


@pytest.mark.parametrize('how', ['script', 'trace', 'fx', 'export', 'vmap', 'compile'])
def test_tables_can_be_recorded_and_transformed(how):
    t = _table()
    f = {'script': lambda: torch.jit.script(t), 'trace': lambda: torch.jit.trace(t, (IDS,)),
         'fx': lambda: torch.fx.symbolic_trace(t),
         'export': lambda: torch.export.export(t, (IDS,)).module(), 'vmap': lambda: torch.vmap(t),
         'compile': lambda: torch.compile(t, backend='eager', fullgraph=True)}[how]()
    assert torch.equal(f(IDS), t.weight[IDS])
    with torch.no_grad():
        t.weight.mul_(2.0)
    if how != 'export':                     # (exported with a copy of the weights)
        assert torch.equal(f(IDS), t.weight[IDS])


def test_operators_refuse_what_they_would_lose():
    """The refusals come before any launch, so they can be seen without a device."""
    import torch.autograd.forward_ad as fw

    from collie_amd import _lib, functional as F, ops
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    ids = torch.zeros(2, dtype=torch.int64)
    calls = [lambda v: F.layer_norm(v), lambda v: F.layer_norm(x, v[0]), lambda v: F.linear(v, w),
             lambda v: F.linear(x, v), lambda v: F.linear(x, v, residual=v[:, :2]),
             lambda v: F.gated_linear(x, w, v), lambda v: F.embedding_rows(v, ids),
             lambda v: ops.embedding_rows_grad(ids, v, 3)]
    for call in calls:
        with fw.dual_level(), pytest.raises(_lib.CollieHipError, match='forward-mode tangent'):
            call(fw.make_dual(x, torch.ones(2, 4)))
        with fw.dual_level(), torch.no_grad(), pytest.raises(_lib.CollieHipError,
                                                             match='forward-mode tangent'):
            call(fw.make_dual(x, torch.ones(2, 4)))
        for transform in (lambda f: torch.func.jvp(f, (x,), (x,)),
                          lambda f: torch.vmap(f)(torch.zeros(5, 2, 4)),
                          lambda f: torch.func.grad(lambda v: f(v).sum())(x),
                          lambda f: torch.jit.trace(f, (x,))):
            with pytest.raises(_lib.CollieHipError, match='vmap, torch.func or torch.jit.trace'):
                transform(call)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode, pytest.raises(_lib.CollieHipError, match='fake tensors'):
        F.layer_norm(mode.from_tensor(x))
