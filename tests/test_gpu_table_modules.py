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


# ---- the tables as modules under torch's transforms ------------------------------------------------
def _table(rows=9, dim=5, **kw):
    from collie_amd import layers
    torch.manual_seed(3)
    t = layers.ScaledEmbedding(rows, dim, **kw).to(DEV)
    with torch.no_grad():
        t.weight.normal_()
    return t


IDS = torch.tensor([[1, 8, 0], [8, 8, 3]])


@pytest.mark.parametrize('frozen', [True, False])
@pytest.mark.parametrize('grad_mode', [True, False])
def test_tables_carry_a_forward_mode_tangent(frozen, grad_mode):
    import torch.autograd.forward_ad as fw
    t = _table()
    t.weight.requires_grad_(not frozen)
    ids, tangent = IDS.to(DEV), torch.randn(9, 5).to(DEV)
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = fw.make_dual(t.weight, tangent)
        y, dy = fw.unpack_dual(torch.func.functional_call(t, {'weight': dual}, (ids,)))
    assert torch.equal(y, t.weight[ids]) and torch.equal(dy, tangent[ids])


@pytest.mark.parametrize('how', ['script', 'trace', 'vmap', 'func_grad', 'jvp', 'compile'])
def test_tables_can_be_recorded_and_transformed(how):
    t = _table()
    t.weight.requires_grad_(False)
    ids = IDS.to(DEV)
    want = t.weight[ids]
    if how == 'script':
        got = torch.jit.script(t)(ids)
    elif how == 'trace':
        traced = torch.jit.trace(t, (ids,))
        torch.empty(1 << 20, device=DEV).fill_(7.0)     # what a recorded allocation might find
        got = traced(ids)
    elif how == 'vmap':
        got = torch.vmap(t)(ids)
    elif how == 'compile':
        got = torch.compile(t, backend='eager', fullgraph=True)(ids)
    else:
        f = lambda w: torch.func.functional_call(t, {'weight': w}, (ids,))      # noqa: E731
        if how == 'func_grad':
            got = torch.func.grad(lambda w: f(w).sum())(t.weight)
            want = torch.bincount(ids.reshape(-1), minlength=9)[:, None].expand(9, 5).float()
        else:
            got, tangent = torch.func.jvp(f, (t.weight,), (2 * t.weight,))
            assert torch.equal(tangent, 2 * want)
    assert torch.equal(got, want)


@pytest.mark.parametrize('padding', [None, 3])
def test_gradients_of_a_table_under_transforms(padding):
    """Batched gradients, gradients of gradients of them, and a tangent that comes from elsewhere, as
    torch.nn.Embedding has them (whole numbers: exact)."""
    import torch.autograd.forward_ad as fw
    own, ref = _table(padding_idx=padding), torch.nn.Embedding(9, 5, padding_idx=padding).to(DEV)
    ids = IDS.to(DEV)
    with torch.no_grad():
        ref.weight.copy_(own.weight.round())
        own.weight.copy_(ref.weight)
    g = torch.Generator().manual_seed(4)
    dys = torch.randint(-3, 4, (4, 2, 3, 5), generator=g).float().to(DEV)
    got = {}
    for name, t in (('own', own), ('ref', ref)):
        y = t(ids)
        (rows,) = torch.autograd.grad(y, [t.weight], dys, is_grads_batched=True, retain_graph=True)
        out = [rows]
        dy = dys[0].clone().requires_grad_()
        (grad,) = torch.autograd.grad(y, [t.weight], dy, create_graph=True)
        (back,) = torch.autograd.grad(grad, [dy], torch.stack([torch.ones_like(grad), grad.detach()]),
                                      is_grads_batched=True)
        out.append(back)
        with fw.dual_level():
            other = fw.make_dual(dys[1], dys[2])
            (grad,) = torch.autograd.grad((t(ids) * other).sum(), [t.weight])
            out += list(fw.unpack_dual(grad))
        got[name] = out
    for a, b in zip(got['own'], got['ref']):
        assert b is not None and torch.equal(a, b)


def test_layers_refuse_gradients_that_stand_for_others():
    from collie_amd import _lib, functional as F
    x, w = torch.ones(3, 4, device=DEV, requires_grad=True), torch.ones(5, 4, device=DEV)
    for y in (F.linear(x, w, activation='silu'), F.gated_linear(x, w, w), F.layer_norm(x)):
        with pytest.raises(RuntimeError, match='vmap, torch.func or torch.jit.trace'):
            torch.autograd.grad(y, [x], torch.ones(2, *y.shape, device=DEV), is_grads_batched=True)
    assert issubclass(_lib.CollieHipError, RuntimeError)


# ---- ids outside a table that is called as a module ------------------------------------------------
@pytest.mark.parametrize('sparse', [False, True])
def test_a_table_reports_ids_outside_of_it(sparse):
    t = _table(sparse=sparse)
    t(IDS.to(DEV))
    t.check_status()
    for bad in (9, -1, 1 << 40):
        ids = torch.tensor([2, bad, 2], device=DEV)
        y = t(ids)
        assert torch.equal(y[[0, 2]], t.weight[[2, 2]]) and torch.equal(y[1], torch.zeros(5, device=DEV))
        with pytest.raises(IndexError, match='outside the table'):
            t.check_status()
        t.check_status()                    # reported once
        y.sum().backward()
        grad = t.weight.grad.to_dense() if sparse else t.weight.grad
        want = torch.zeros(9, 5, device=DEV)
        want[2] = 2.0
        assert torch.equal(grad, want)
        t.weight.grad = None
        t._status.zero_()
    assert set(t.state_dict()) == {'weight'}


def test_a_model_reports_ids_outside_tables_that_it_calls():
    from collie_amd.model import MatrixFactorizationModel

    class Shape:
        num_users, num_items, num_negative_samples = 30, 20, 1

    class Sum(MatrixFactorizationModel):
        def forward(self, users, items):
            return (self.user_embeddings(users) * self.item_embeddings(items)).sum(1)

    model = Sum(train=Shape(), embedding_dim=8, lr_scheduler_func=None).to(DEV)
    good, bad = torch.tensor([0, 19], device=DEV), torch.tensor([0, 20], device=DEV)
    model(good, good)
    model.check_status()
    model(bad, bad)                         # 20 is a user, but no item
    with pytest.raises(IndexError, match='outside the table'):
        model.check_status()
    model.check_status()


def test_a_table_captured_before_its_first_call():
    t = _table()
    t.weight.requires_grad_(False)
    ids = IDS.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = t(ids)
    assert t._status is None
    for shift in range(3):
        ids.copy_((IDS + shift) % 9)
        graph.replay()
        assert torch.equal(y, t.weight[ids])
        torch.cuda.synchronize()


def test_a_table_first_called_in_inference_mode():
    from collie_amd import layers
    t = layers.ScaledEmbedding(5, 3).to(DEV)
    with torch.inference_mode():
        y = t(torch.tensor([1, 7], device=DEV))
    assert torch.equal(y[1], torch.zeros(3, device=DEV))
    for _ in range(2):
        with pytest.raises(IndexError):
            t.check_status()
        t(torch.tensor([-1], device=DEV))


def test_tables_past_the_limits_of_the_entry_points_are_torch_s():
    t = _table(rows=2, dim=(1 << 20) + 1)
    ids = torch.tensor([1, 0, 1], device=DEV)
    y = t(ids)
    assert torch.equal(y, t.weight[ids])
    y.sum().backward()
    assert torch.equal(t.weight.grad[:, :2].cpu(), torch.tensor([[1.0, 1.0], [2.0, 2.0]]))


def test_layers_inside_a_compiled_function():
    """The compiler breaks its graph at the functions and calls them as they are."""
    from collie_amd import functional as F
    w = torch.randn(6, 4, generator=torch.Generator().manual_seed(0)).to(DEV).requires_grad_()
    x = torch.randn(9, 4, generator=torch.Generator().manual_seed(1)).to(DEV)

    def f(x, w):
        return F.linear(F.layer_norm(x * 2.0), w, activation='silu') + 1.0

    got = torch.compile(f, backend='eager')(x, w)
    want = f(x, w)
    assert torch.equal(got, want)
    (a,), (b,) = (torch.autograd.grad(y.sum(), [w]) for y in (got, want))
    assert torch.equal(a, b)
