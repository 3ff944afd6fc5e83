"""
GPU tests (``-m gpu``) of the ranking-head operators (``collie_amd.functional``): every result and
gradient against float64 within the bounds of ``head_bounds``, at the sizes, strides and inputs where
a kernel can go wrong; capture and replay; equal bits from equal calls; and the modules together.
"""
import pytest
import torch

import head_bounds as hb

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def leaf(t, grad=True):
    return None if t is None else t.to(DEV).requires_grad_(grad)


def f64(t):
    return None if t is None else t.double()


# ---- embedding rows ------------------------------------------------------------------------------
EMBED = [
    # rows, dim, n, distribution
    (1, 1, 1, 'uniform'), (7, 3, 5, 'uniform'), (50, 64, 64, 'uniform'), (50, 64, 65, 'one'),
    (300, 20, 4096, 'uniform'), (300, 33, 4097, 'skew'), (5, 16, 20000, 'uniform'),
    (1, 8, 9000, 'one'), (100000, 12, 6000, 'uniform'), (70, 1000, 700, 'skew'),
    (40, 2049, 130, 'skew'), (3000, 128, 30000, 'skew'), (200000, 1, 50000, 'skew'),
]


def make_ids(rows, n, kind, seed):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(n, generator=g)
    if kind == 'one':
        return torch.full((n,), rows // 2, dtype=torch.int64)
    return ((u ** 6 if kind == 'skew' else u) * rows).long().clamp_(0, rows - 1)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,dim,n,kind', EMBED)
def test_embedding_rows(rows, dim, n, kind, dtype):
    from collie_amd import functional as F
    ids = make_ids(rows, n, kind, rows + n)
    w, dy = rand((rows, dim), dtype, 1), rand((n, dim), dtype, 2)
    scale = 1.0 if n % 2 else 2.5
    weight = leaf(w)
    y = F.embedding_rows(weight, ids.to(DEV).to(torch.int32 if n % 3 == 0 else torch.int64),
                         scale=scale)
    want = w.double()[ids] * scale
    hb.check(y.detach(), want, hb.F * want.abs(), dtype)
    (grad,) = torch.autograd.grad(y, [weight], dy.to(DEV))
    total = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids, dy.double()) * scale
    mag = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids, dy.double().abs()) * scale
    count = torch.bincount(ids, minlength=rows).double().unsqueeze(1)
    hb.check(grad, total, (count + 2) * hb.F * mag, dtype)
    assert (grad.cpu()[count.reshape(-1) == 0] == 0).all()
    again = torch.autograd.grad(F.embedding_rows(weight, ids.to(DEV), scale=scale), [weight],
                                dy.to(DEV))[0]
    assert torch.equal(grad, again)


def test_embedding_rows_bad_ids_padding_shapes_and_strides():
    from collie_amd import functional as F
    w = rand((10, 6), torch.float32, 3)
    ids = torch.tensor([[0, 9, 10], [-1, 4, 4], [1 << 40, 3, 0]])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    weight = leaf(w)
    y = F.embedding_rows(weight, ids.to(DEV), status=status, padding_idx=4)
    assert status.item() == 1
    bad = (ids < 0) | (ids >= 10)
    want = torch.where(bad.unsqueeze(-1), torch.zeros(6), w[ids.clamp(0, 9)])
    assert torch.equal(y.detach().cpu(), want)
    (grad,) = torch.autograd.grad(y.sum(), [weight])        # an expanded dy
    ref = torch.zeros(10, 6)
    for r in (0, 9, 3, 0):
        ref[r] += 1
    assert torch.equal(grad.cpu(), ref)
    # transposed ids, dy with rows apart, a table that is a view with an odd offset
    table = rand((21, 5), torch.bfloat16, 4).to(DEV)[1:].requires_grad_()
    idt = torch.arange(12).reshape(3, 4).to(DEV).t()
    y = F.embedding_rows(table, idt)
    dy = rand((12, 9), torch.bfloat16, 5).to(DEV)[:, 2:7]
    (grad,) = torch.autograd.grad(y, [table], dy.reshape(4, 3, 5))
    ref = torch.zeros(20, 5, dtype=torch.bfloat16)
    ref[idt.cpu().reshape(-1)] = dy.cpu()
    assert torch.equal(grad.cpu(), ref)
    from collie_amd import ops
    grad = ops.embedding_rows_grad(idt.reshape(-1), dy, 20)
    assert torch.equal(grad.cpu(), ref)
    # nothing looked up
    empty = F.embedding_rows(table, torch.empty(0, 2, dtype=torch.int64, device=DEV))
    assert empty.shape == (0, 2, 5)
    assert torch.equal(torch.autograd.grad(empty.sum(), [table])[0], torch.zeros_like(table))


def test_embedding_rows_second_derivative_and_sparse_gradient():
    from collie_amd import functional as F
    w = leaf(rand((6, 4), torch.float32, 6))
    ids = torch.tensor([5, 1, 1, 2], device=DEV)
    y = F.embedding_rows(w, ids, scale=0.5)
    (g,) = torch.autograd.grad((y ** 2).sum(), [w], create_graph=True)
    (gg,) = torch.autograd.grad((g ** 2).sum(), [w])
    w64 = w.detach().cpu().double().requires_grad_()
    y64 = w64[ids.cpu()] * 0.5
    (g64,) = torch.autograd.grad((y64 ** 2).sum(), [w64], create_graph=True)
    (gg64,) = torch.autograd.grad((g64 ** 2).sum(), [w64])
    # every value passes through fewer than 8 roundings
    torch.testing.assert_close(gg.double().cpu(), gg64, rtol=8 * hb.F, atol=0)
    y = F.embedding_rows(w, ids, scale=0.5, sparse=True, padding_idx=2)
    (sp,) = torch.autograd.grad(y.sum(), [w])
    assert sp.is_sparse
    ref = torch.zeros(6, 4)
    ref[5], ref[1] = 0.5, 1.0
    assert torch.equal(sp.to_dense().cpu(), ref)


def test_layers_other_than_the_rows_refuse_a_second_derivative():
    from collie_amd import functional as F
    x, w, b = (leaf(rand(s, torch.float32, i)) for i, s in enumerate([(3, 4), (5, 4), (5,)]))
    for y in (F.linear(x, w, b, 'silu'), F.gated_linear(x, w, w), F.layer_norm(x, w[0], w[1])):
        (g,) = torch.autograd.grad(y.sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match='differentiated once'):
            torch.autograd.grad(g.sum(), [x])
    # only what is asked for is computed, and a residual's gradient may be differentiated again
    r = leaf(rand((3, 5), torch.float32, 4))
    y = F.linear(x.detach(), w.detach(), residual=r)
    (g,) = torch.autograd.grad((y ** 2).sum(), [r], create_graph=True)
    assert torch.equal(torch.autograd.grad(g.sum(), [r])[0], torch.full_like(r, 2.0))
    y = F.linear(x, w, b, 'gelu', r)
    every = torch.autograd.grad(y, [x, w, b, r], torch.ones_like(y), retain_graph=True)
    for leaf_of, g in zip((x, w, b, r), every):
        (one,) = torch.autograd.grad(y, [leaf_of], torch.ones_like(y), retain_graph=True)
        assert torch.equal(one, g)


def test_embedding_status_may_be_cleared_between_the_passes():
    from collie_amd import functional as F
    w = leaf(rand((6, 4), torch.float32, 6))
    ids = torch.tensor([5, 6, -1, 2], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = F.embedding_rows(w, ids, status=status)
    assert status.item() == 1
    status.zero_()
    (g,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert status.item() == 1
    ref = torch.zeros(6, 4)
    ref[5], ref[2] = 1.0, 1.0
    assert torch.equal(g.cpu(), ref)


@pytest.mark.parametrize('cls', ['ScaledEmbedding', 'ZeroEmbedding'])
@pytest.mark.parametrize('sparse', [False, True])
def test_table_modules_give_what_torch_gives(cls, sparse):
    from collie_amd import layers
    torch.manual_seed(0)
    t = getattr(layers, cls)(20, 7, sparse=sparse, padding_idx=3).to(DEV)
    with torch.no_grad():
        t.weight.copy_(torch.randn(20, 7))
    ids = torch.tensor([[1, 3, 3], [19, 0, 1]], device=DEV)
    y = t(ids)
    ref = torch.nn.functional.embedding(ids.cpu(), t.weight.detach().cpu())
    assert torch.equal(y.detach().cpu(), ref)
    y.sum().backward()
    want = torch.zeros(20, 7)
    want[1], want[19], want[0] = 2, 1, 1
    assert t.weight.grad.is_sparse == sparse
    assert torch.equal((t.weight.grad.to_dense() if sparse else t.weight.grad).cpu(), want)


@pytest.mark.parametrize('n', [0, 1000, 70000])
@pytest.mark.parametrize('dim', [1, 24])
def test_dense_table_gradients_of_the_models(n, dim):
    """Few rows by atomic adds, many by sorted ids: the same sums."""
    from collie_amd import functional as F
    assert n < F.SORTED_GRAD_ROWS or n > F.SORTED_GRAD_ROWS
    ids, vals = make_ids(500, n, 'skew', 3).int(), rand((n, dim), torch.float32, 4)
    table = torch.zeros(500, dim, device=DEV)
    got = F.table_grad(table, ids.to(DEV), vals.to(DEV))
    want = torch.zeros(500, dim, dtype=torch.float64).index_add_(0, ids, vals.double())
    mag = torch.zeros(500, dim, dtype=torch.float64).index_add_(0, ids, vals.double().abs())
    hb.check(got, want, (torch.bincount(ids, minlength=500)[:, None] + 2) * hb.F * mag,
             torch.float32)


def test_generic_route_of_a_dense_model_on_a_large_batch():
    from collie_amd.model import MatrixFactorizationModel

    class Shape:
        num_users, num_items, num_negative_samples = 300, 200, 1

    torch.manual_seed(0)
    model = MatrixFactorizationModel(train=Shape(), embedding_dim=16, sparse=False,
                                     lr_scheduler_func=None).to(DEV)
    with torch.no_grad():
        for t in (model.user_embeddings, model.item_embeddings):
            t.weight.copy_(torch.randn(t.weight.shape))
    users, items = make_ids(300, 70000, 'skew', 5), make_ids(200, 70000, 'skew', 6)
    c = rand((70000,), torch.float32, 7)
    (model(users.to(DEV), items.to(DEV)) * c.to(DEV)).sum().backward()
    rows = {'user_embeddings': (users, model.item_embeddings.weight.detach().cpu()[items]),
            'item_embeddings': (items, model.user_embeddings.weight.detach().cpu()[users]),
            'user_biases': (users, torch.ones(70000, 1)), 'item_biases': (items, torch.ones(70000, 1))}
    for name, (ids, other) in rows.items():
        table = getattr(model, name).weight
        vals = c.double()[:, None] * other.double()
        want = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, ids, vals)
        mag = torch.zeros(table.shape, dtype=torch.float64).index_add_(0, ids, vals.abs())
        count = torch.bincount(ids, minlength=table.shape[0])[:, None]
        hb.check(table.grad, want, (count + 4) * hb.F * mag, torch.float32)


# ---- layer norm ----------------------------------------------------------------------------------
NORM = [(1, 1), (1, 128), (3, 5), (17, 64), (130, 65), (64, 128), (33, 255), (9, 256), (70, 511),
        (20, 1000), (40, 1023), (5, 1025), (6, 2048), (11, 3001), (4, 4096), (3, 8191), (2, 8192),
        (3, 8193), (2, 20011), (5000, 16)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,dim', NORM)
def test_layer_norm(rows, dim, dtype):
    from collie_amd import functional as F
    x = rand((rows, dim), dtype, dim) * 2 + 1
    w, b = 1 + rand((dim,), dtype, 2, 0.2), rand((dim,), dtype, 3)
    dy = rand((rows, dim), dtype, 4)
    leaves = [leaf(t) for t in (x, w, b)]
    y = F.layer_norm(*leaves)
    got = [y.detach()] + list(torch.autograd.grad(y, leaves, dy.to(DEV)))
    ref = hb.layer_norm(f64(x), f64(w), f64(b), 1e-5, f64(dy), dtype)
    for g, name in zip(got, ('y', 'dx', 'dw', 'db')):
        hb.check(g, *ref[name], dtype)
    again = torch.autograd.grad(F.layer_norm(*leaves), leaves, dy.to(DEV))
    assert all(torch.equal(a, g) for a, g in zip(again, got[1:]))
    with torch.no_grad():
        assert torch.equal(F.layer_norm(*leaves), got[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_layer_norm_parameters_strides_and_missing_parts(dtype):
    from collie_amd import functional as F
    base = rand((2, 9, 45), dtype, 7).to(DEV)
    x = base[0, :, 3:43]                                    # rows 45 apart, an odd offset
    dy = rand((9, 41), dtype, 8).to(DEV)[:, 1:]
    ones, zeros = torch.ones(40).double(), torch.zeros(40).double()
    w32, b32 = 1 + rand((40,), torch.float32, 9, 0.2), rand((40,), torch.float32, 10)
    for w, b in ((None, None), (w32, None), (None, b32), (w32, b32)):
        xs, ws, bs = x.detach().requires_grad_(), leaf(w), leaf(b)
        leaves = [t for t in (xs, ws, bs) if t is not None]
        y = F.layer_norm(xs, ws, bs, eps=1e-3)
        grads = torch.autograd.grad(y, leaves, dy)
        ref = hb.layer_norm(f64(x.cpu()), ones if w is None else f64(w),
                            zeros if b is None else f64(b), 1e-3, f64(dy.cpu()), dtype)
        hb.check(y.detach(), *ref['y'], dtype)
        names = ['dx'] + ['dw'] * (w is not None) + ['db'] * (b is not None)
        for g, name in zip(grads, names):
            hb.check(g, *ref[name], dtype if name == 'dx' else torch.float32)
    # only some gradients wanted; three dimensions; no rows
    ws = leaf(w32)
    y = F.layer_norm(base.reshape(2, 9, 45)[..., :40], ws)
    assert y.shape == (2, 9, 40)
    (dw,) = torch.autograd.grad(y, [ws], torch.ones_like(y))
    ref = hb.layer_norm(f64(base.cpu()[..., :40].reshape(18, 40)), f64(w32), zeros, 1e-5,
                        torch.ones(18, 40).double(), dtype)
    hb.check(dw, *ref['dw'], torch.float32)
    empty = torch.empty(0, 40, dtype=dtype, device=DEV, requires_grad=True)
    y = F.layer_norm(empty, ws)
    dx, dw = torch.autograd.grad(y.sum(), [empty, ws])
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_constant_rows_and_non_finite_values():
    from collie_amd import functional as F
    x = torch.full((4, 300), 1000.0)
    y = F.layer_norm(x.to(DEV))
    assert torch.equal(y.cpu(), torch.zeros(4, 300))        # 300 x 1000 is exact in float32
    x[1, 5], x[2, 7] = float('inf'), float('nan')
    y = F.layer_norm(x.to(DEV)).cpu()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    assert torch.equal(y[[0, 3]], torch.zeros(2, 300))      # neighbours are not touched


# ---- linear and gated layers ---------------------------------------------------------------------
ACTS = ['identity', 'relu', 'leaky_relu', 'sigmoid', 'silu', 'gelu']
SHAPES = [
    # rows, n_in, n_out
    (1, 1, 1), (1, 64, 128), (2, 33, 17), (5, 1024, 96), (16, 509, 130), (17, 128, 64),
    (64, 40, 72), (65, 129, 255), (100, 8, 8), (129, 256, 128), (200, 300, 40), (257, 64, 264),
    (300, 16, 513), (1000, 24, 1), (1, 2048, 3), (700, 128, 128), (1030, 72, 200), (4100, 64, 32),
]


def run_linear(m, n_in, n_out, dtype, kind, bias, residual, seed=0):
    from collie_amd import functional as F
    x, w = rand((m, n_in), dtype, seed + 1), rand((n_out, n_in), dtype, seed + 2, n_in ** -0.5)
    b = rand((n_out,), dtype, seed + 3) if bias else None
    r = rand((m, n_out), dtype, seed + 4) if residual else None
    dy = rand((m, n_out), dtype, seed + 5)
    leaves = [leaf(t) for t in (x, w, b, r)]
    y = F.linear(*leaves[:3], activation=kind, residual=leaves[3])
    there = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, there, dy.to(DEV))
    ref = hb.linear(f64(x), f64(w), f64(b), f64(r), kind, f64(dy), dtype)
    hb.check(y.detach(), *ref['y'], dtype)
    hb.check(grads[0], *ref['dx'], dtype)
    hb.check(grads[1], *ref['dw'], dtype)
    if bias:
        hb.check(grads[2], *ref['db'], dtype)
    if residual:
        assert torch.equal(grads[-1].cpu(), dy)
    with torch.no_grad():
        assert torch.equal(F.linear(*leaves[:3], activation=kind, residual=leaves[3]), y)
    again = torch.autograd.grad(F.linear(*leaves[:3], activation=kind, residual=leaves[3]), there,
                                dy.to(DEV))
    assert all(torch.equal(a, g) for a, g in zip(again, grads))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('i', range(len(SHAPES)))
def test_linear(i, dtype):
    m, n_in, n_out = SHAPES[i]
    run_linear(m, n_in, n_out, dtype, ACTS[i % 6], i % 3 != 0, i % 2 == 0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ACTS)
def test_linear_activations(kind, dtype):
    run_linear(37, 48, 56, dtype, kind, True, False, seed=20)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ACTS)
def test_activations_over_their_whole_range(kind, dtype):
    """One input, weight one: z runs through the range, so every activation meets its ends."""
    from collie_amd import functional as F
    z = torch.cat([torch.linspace(-300, 300, 4801), torch.linspace(-3e4, 3e4, 101),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-5])]).to(dtype).reshape(-1, 1)
    one, dy = torch.ones(1, 1, dtype=dtype), torch.ones_like(z)
    x, w = leaf(z), leaf(one)
    y = F.linear(x, w, activation=kind)
    dx, dw = torch.autograd.grad(y, [x, w], dy.to(DEV))
    ref = hb.linear(f64(z), f64(one), None, None, kind, f64(dy), dtype)
    hb.check(y.detach(), *ref['y'], dtype)
    hb.check(dx, *ref['dx'], dtype)
    hb.check(dw, *ref['dw'], dtype)
    y = F.gated_linear(x, w, w, activation=kind)
    dx, dwg = torch.autograd.grad(y, [x, w], dy.to(DEV))
    if dtype != torch.float16:      # (z^2 is past float16's range)
        ref = hb.gated(f64(z), f64(one), f64(one), None, None, kind, f64(dy), dtype)
        hb.check(y.detach(), *ref['y'], dtype)
        hb.check(dx, *ref['dx'], dtype)


def run_gated(m, n_in, n_out, dtype, kind, bias, seed=0):
    from collie_amd import functional as F
    std = n_in ** -0.5
    x = rand((m, n_in), dtype, seed + 1)
    wg, wu = rand((n_out, n_in), dtype, seed + 2, std), rand((n_out, n_in), dtype, seed + 3, std)
    bg, bu = (rand((n_out,), dtype, seed + s) if bias else None for s in (4, 5))
    dy = rand((m, n_out), dtype, seed + 6)
    leaves = [leaf(t) for t in (x, wg, wu, bg, bu)]
    there = [t for t in leaves if t is not None]
    y = F.gated_linear(*leaves, activation=kind)
    grads = torch.autograd.grad(y, there, dy.to(DEV))
    ref = hb.gated(f64(x), f64(wg), f64(wu), f64(bg), f64(bu), kind, f64(dy), dtype)
    hb.check(y.detach(), *ref['y'], dtype)
    for g, name in zip(grads, ('dx', 'dwg', 'dwu', 'dbg', 'dbu')):
        hb.check(g, *ref[name], dtype)
    with torch.no_grad():
        assert torch.equal(F.gated_linear(*leaves, activation=kind), y)
    again = torch.autograd.grad(F.gated_linear(*leaves, activation=kind), there, dy.to(DEV))
    assert all(torch.equal(a, g) for a, g in zip(again, grads))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('i', range(len(SHAPES)))
def test_gated(i, dtype):
    m, n_in, n_out = SHAPES[i]
    run_gated(m, n_in, n_out, dtype, ACTS[(i + 4) % 6], i % 2 == 0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ACTS)
def test_gated_activations(kind, dtype):
    run_gated(37, 48, 56, dtype, kind, True, seed=30)


# enough 256 x 256 tiles for the large-tile kernel in the forward pass, in dx and in dW
LARGE = [(4200, 72, 4104), (4200, 4104, 72), (72, 4104, 4200), (4111, 77, 4099)]


@pytest.mark.parametrize('dtype', TYPES[1:])
@pytest.mark.parametrize('m,n_in,n_out', LARGE)
def test_large_tiles(m, n_in, n_out, dtype):
    run_linear(m, n_in, n_out, dtype, 'gelu', True, True, seed=40)
    run_gated(m, n_in, n_out // 2 + 1, dtype, 'silu', True, seed=50)


@pytest.mark.parametrize('dtype', TYPES)
def test_layers_take_strides_more_dimensions_and_no_rows(dtype):
    from collie_amd import functional as F
    base = rand((4, 6, 70), dtype, 11).to(DEV)
    x = base[..., 1:52]
    w, w2 = rand((19, 51), dtype, 12, 0.15), rand((51, 19), dtype, 13, 0.15)
    b = rand((19,), dtype, 14)
    dy = rand((4, 6, 19), dtype, 15)
    ws = [leaf(w), w2.to(DEV).t().requires_grad_(), leaf(b)]
    xs = x.detach().requires_grad_()
    y = F.linear(xs, ws[0], ws[2], 'silu')
    grads = torch.autograd.grad(y, [xs, ws[0], ws[2]], dy.to(DEV))
    flat = f64(x.cpu().reshape(24, 51))
    ref = hb.linear(flat, f64(w), f64(b), None, 'silu', f64(dy.reshape(24, 19)), dtype)
    for g, name in zip([y.detach(), *grads], ('y', 'dx', 'dw', 'db')):
        val, bound = ref[name]
        shape = g.shape
        hb.check(g, val.reshape(shape), bound.reshape(shape), dtype)
    # a transposed weight, rows apart without a copy, a scalar-like dy
    x2 = base.reshape(24, 70)[:, 2:53].detach().requires_grad_()
    y = F.gated_linear(x2, ws[0], ws[1], activation='sigmoid')
    grads = torch.autograd.grad(y.sum(), [x2, ws[0], ws[1]])
    ref = hb.gated(f64(x2.detach().cpu()), f64(w), f64(w2.t()), None, None, 'sigmoid',
                   torch.ones(24, 19).double(), dtype)
    for g, name in zip([y.detach(), *grads], ('y', 'dx', 'dwg', 'dwu')):
        hb.check(g, *ref[name], dtype)
    empty = torch.empty(0, 51, dtype=dtype, device=DEV, requires_grad=True)
    for y in (F.linear(empty, ws[0], ws[2], 'gelu'), F.gated_linear(empty, ws[0], ws[1])):
        assert y.shape == (0, 19)
        dx, dw = torch.autograd.grad(y.sum(), [empty, ws[0]])
        assert dx.shape == (0, 51) and torch.equal(dw, torch.zeros_like(dw))
    # one gradient at a time
    full = torch.autograd.grad(F.linear(xs, ws[0], ws[2], 'gelu'), [xs, ws[0], ws[2]], dy.to(DEV))
    for k in range(3):
        args = [t.detach() for t in (xs, ws[0], ws[2])]
        args[k] = args[k].requires_grad_()
        (g,) = torch.autograd.grad(F.linear(*args, 'gelu'), [args[k]], dy.to(DEV))
        assert torch.equal(g, full[k])


def test_layers_large_values():
    """float16 pre-activations beyond its range leave finite gradients; infinities stay in their
    rows."""
    from collie_amd import functional as F
    x = torch.full((2, 64), 200.0, dtype=torch.float16)
    w = torch.full((8, 64), 10.0, dtype=torch.float16)
    xs, ws = leaf(x), leaf(-w)
    y = F.linear(xs, ws, activation='silu')                 # z = -128,000
    assert torch.equal(y.detach().cpu(), torch.zeros(2, 8).half())
    dx, dw = torch.autograd.grad(y, [xs, ws], torch.ones_like(y))
    assert torch.equal(dx.cpu(), torch.zeros(2, 64).half())
    assert torch.equal(dw.cpu(), torch.zeros(8, 64).half())
    for dtype in TYPES:
        a = rand((40, 96), dtype, 16)
        a[3, 7] = float('inf')
        a[21, 95] = float('nan')
        b = rand((24, 96), dtype, 17).abs() + 0.1
        y = F.linear(a.to(DEV), b.to(DEV)).cpu()
        assert torch.isinf(y[3]).all() and torch.isnan(y[21]).all()
        keep = [i for i in range(40) if i not in (3, 21)]
        assert torch.isfinite(y[keep]).all()


def test_float32_products_with_values_that_have_no_finite_parts():
    """float32 products are made of bfloat16 parts; tiles with values that have none (infinities, NaN,
    the top of the range) are computed again as they are.  Enough tiles that a workgroup works on
    several: the others, before and after, stay what they are."""
    from collie_amd import functional as F
    a, b = rand((5200, 72), torch.float32, 70), rand((2600, 72), torch.float32, 71)
    a[300, 5], a[1111, 70], a[5199, 0] = float('inf'), float('nan'), -float('inf')
    a[2000] = 0.0
    a[2000, 3] = 3.4e38                     # rounds up to no finite bfloat16
    b[17] = 0.0
    b[17, 3] = 0.5
    y = F.linear(a.to(DEV), b.to(DEV)).cpu()
    assert torch.isnan(y[1111]).all()
    for row in (300, 5199):
        k = 5 if row == 300 else 0
        want = a[row, k] * b[:, k]          # +-inf by the sign of b, NaN where b is 0
        assert torch.equal(torch.nan_to_num(y[row]), torch.nan_to_num(want))
    assert y[2000, 17].item() == a[2000, 3].item() * 0.5
    keep = torch.ones(5200, dtype=torch.bool)
    keep[[300, 1111, 5199, 2000]] = False
    val, bound = hb.product(a[keep].double(), b.double())
    hb.check(y[keep], val, bound, torch.float32)
    # the same through the gradients: dx has the bad rows, dW the bad columns, all of it
    x, w = leaf(a), leaf(b)
    dy = rand((5200, 2600), torch.float32, 72).to(DEV)
    dx, dw = torch.autograd.grad(F.linear(x, w), [x, w], dy)
    val, bound = hb.product(dy.cpu().double(), b.double().T)
    hb.check(dx, val, bound, torch.float32)
    good = [k for k in range(72) if k not in (0, 3, 5, 70)]
    val, bound = hb.product(dy.cpu().double().T, a[:, good].double().T)
    hb.check(dw[:, good], val, bound, torch.float32)
    assert torch.isnan(dw[:, 70]).all() and torch.isinf(dw[:, [0, 5]]).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_gradients_against_differences(dtype):
    """Directional derivatives of a loss through all operators, in float64 differences of the plain
    formula around the same point: 64 * (half a step) relative to the sum of magnitudes covers the
    at most a dozen roundings of every path."""
    from collie_amd import functional as F
    ids = torch.tensor([3, 1, 4, 1, 5, 9, 2, 6, 5, 3])
    shapes = {'e': (10, 24), 'nw': (24,), 'nb': (24,), 'g': (40, 24), 'u': (40, 24), 'd': (24, 40)}
    p = {k: rand(s, dtype, 40 + i, 0.3) for i, (k, s) in enumerate(shapes.items())}
    c = rand((10, 24), dtype, 50)

    def plain(q):
        x = q['e'][ids] * 2.0
        xc = x - x.mean(1, keepdim=True)
        h = xc * ((xc * xc).mean(1, keepdim=True) + 1e-5).rsqrt() * q['nw'] + q['nb']
        g = h @ q['g'].T
        y = (g * torch.sigmoid(g) * (h @ q['u'].T)) @ q['d'].T + x
        return (y * c.double()).sum()

    q = {k: leaf(v) for k, v in p.items()}
    x = F.embedding_rows(q['e'], ids.to(DEV), scale=2.0)
    h = F.layer_norm(x, q['nw'], q['nb'])
    y = F.linear(F.gated_linear(h, q['g'], q['u']), q['d'], residual=x)
    grads = dict(zip(q, torch.autograd.grad(y, list(q.values()), c.to(DEV))))
    p64 = {k: v.double() for k, v in p.items()}
    for k in p:
        direction = rand(shapes[k], torch.float32, 60).double()
        step = 1e-5
        up, down = ({**p64, k: p64[k] + s * step * direction} for s in (1, -1))
        slope = ((plain(up) - plain(down)) / (2 * step)).item()
        terms = grads[k].double().cpu() * direction
        room = 64 * hb.U[dtype] * terms.abs().sum().item() + 1e-6 * abs(slope)
        assert abs(terms.sum().item() - slope) <= room, (k, terms.sum().item(), slope, room)


def block(dim, hidden, dtype):
    from collie_amd import layers
    torch.manual_seed(5)
    m = torch.nn.ModuleDict({
        'table': layers.ScaledEmbedding(50, dim), 'norm': layers.LayerNorm(dim),
        'gated': layers.GatedLinear(dim, hidden), 'back': layers.Linear(hidden, dim),
        'head': layers.Linear(dim, 1, activation='sigmoid')}).to(DEV, dtype)
    with torch.no_grad():
        m['table'].weight.mul_(50)
    return m


def through(m, ids):
    x = m['table'](ids)
    return m['head'](m['back'](m['gated'](m['norm'](x)), residual=x))


@pytest.mark.parametrize('dtype', TYPES)
def test_operators_together_as_a_block_that_trains(dtype):
    m = block(40, 72, dtype)
    ref = torch.nn.ModuleDict({
        'table': torch.nn.Embedding(50, 40), 'norm': torch.nn.LayerNorm(40),
        'gate': torch.nn.Linear(40, 72), 'up': torch.nn.Linear(40, 72),
        'back': torch.nn.Linear(72, 40), 'head': torch.nn.Linear(40, 1)}).double()
    names = {f'gated.{k}.{p}': f'{k}.{p}' for k in ('gate', 'up') for p in ('weight', 'bias')}
    own = dict(m.named_parameters())
    with torch.no_grad():
        for k, v in own.items():
            dict(ref.named_parameters())[names.get(k, k)].copy_(v)
    ids = torch.randint(0, 50, (33,), generator=torch.Generator().manual_seed(1))
    c = rand((33, 1), torch.float32, 2)
    (through(m, ids.to(DEV)) * c.to(DEV).to(dtype)).sum().backward()
    x = ref['table'](ids)
    h = ref['norm'](x)
    h = torch.nn.functional.silu(ref['gate'](h)) * ref['up'](h)
    (torch.sigmoid(ref['head'](ref['back'](h) + x)) * c.to(dtype).double()).sum().backward()
    theirs = dict(ref.named_parameters())
    for k, v in own.items():
        a, b = v.grad.double().cpu(), theirs[names.get(k, k)].grad
        # at most 16 roundings on any path from the loss to a gradient, in the 2-norm
        assert (a - b).norm() <= 16 * hb.U[dtype] * b.norm(), k
    torch.optim.SGD(m.parameters(), lr=0.1).step()
    assert torch.isfinite(through(m, ids.to(DEV))).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_capture_and_replay_forward_and_backward(dtype):
    """A whole training pass as one graph, replayed on new inputs with eager work in between."""
    m = block(64, 96, dtype)
    params = list(m.parameters())
    ids = torch.zeros(5000, dtype=torch.int64, device=DEV)
    c = torch.zeros(5000, 1, dtype=dtype, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(through(m, ids), params, c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = through(m, ids)
        out = [y.detach(), *torch.autograd.grad(y, params, c)]
    del y       # the captured autograd graph: its nodes belong to the capture's stream
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(0, 50, (5000,), generator=g).to(DEV))
        c.copy_(rand((5000, 1), dtype, seed).to(DEV))
        graph.replay()
        replayed = [t.clone() for t in out]
        y2 = through(m, ids)
        eager = [y2, *torch.autograd.grad(y2, params, c)]
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b.detach())


def test_another_stream_gives_the_same():
    m = block(64, 96, torch.float32)
    params = list(m.parameters())
    ids = torch.arange(3000, device=DEV) % 50
    y = through(m, ids)
    first = torch.autograd.grad(y, params, torch.ones_like(y))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = through(m, ids)
        second = torch.autograd.grad(y, params, torch.ones_like(y))
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


# ---- the hybrid model's head with residual blocks ------------------------------------------------
def deep_hybrid(freeze, **kw):
    from collie_amd.hybrid import HybridPretrainedModel
    from collie_amd.model import MatrixFactorizationModel

    class Shape:
        num_users, num_items, num_negative_samples = 60, 40, 3

    torch.manual_seed(2)
    mf = MatrixFactorizationModel(train=Shape(), embedding_dim=10, lr_scheduler_func=None)
    with torch.no_grad():
        for t in (mf.user_embeddings, mf.item_embeddings, mf.user_biases, mf.item_biases):
            t.weight.copy_(torch.randn(t.weight.shape))
    model = HybridPretrainedModel(train=Shape(), item_metadata=torch.randn(40, 7),
                                  user_metadata=torch.randn(60, 5), trained_model=mf,
                                  item_metadata_layers_dims=[9], combined_layers_dims=[24, 12],
                                  combined_blocks=2, freeze_embeddings=freeze,
                                  lr_scheduler_func=None, **kw)
    return model.to(DEV)


def deep_reference(model, users, items):
    """The same head in float64 torch on the CPU; returns (scores, {name: leaf})."""
    p = {k: v.detach().cpu().double().requires_grad_(v.requires_grad)
         for k, v in model.named_parameters()}

    def lin(x, name):
        return x @ p[name + '.weight'].T + p[name + '.bias']

    leaky = torch.nn.functional.leaky_relu
    x = torch.cat([model.user_metadata.cpu().double()[users], p['embeddings.0.weight'][users],
                   p['embeddings.1.weight'][items],
                   leaky(lin(model.item_metadata.cpu().double()[items], 'item_metadata_layer_0'))], 1)
    x = leaky(lin(x, 'combined_layer_0'))
    for i in range(2):
        b = f'combined_block_{i}.'
        h = torch.nn.functional.layer_norm(x, (24,), p[b + 'norm.weight'], p[b + 'norm.bias'])
        h = torch.nn.functional.silu(lin(h, b + 'gated.gate')) * lin(h, b + 'gated.up')
        x = lin(h, b + 'back') + x
    x = leaky(lin(x, 'combined_layer_1'))
    s = lin(x, 'combined_layer_2')[:, 0]
    return s + p['biases.0.weight'][users, 0] + p['biases.1.weight'][items, 0], p


@pytest.mark.parametrize('freeze', [True, False])
def test_hybrid_head_with_blocks(freeze):
    model = deep_hybrid(freeze, loss='bpr', optimizer='adam')
    g = torch.Generator().manual_seed(9)
    users, items = torch.randint(0, 60, (333,), generator=g), torch.randint(0, 40, (333,), generator=g)
    c = rand((333,), torch.float32, 10)
    scores = model(users.to(DEV), items.to(DEV))
    (scores * c.to(DEV)).sum().backward()
    want, p = deep_reference(model, users, items)
    (want * c.double()).sum().backward()
    # sixteen layers of at most 48 terms: their float32 roundings, in the 2-norm
    room = 16 * 48 * hb.F
    assert (scores.detach().cpu().double() - want).norm() <= room * want.norm()
    for k, v in model.named_parameters():
        if v.requires_grad:
            assert (v.grad.cpu().double() - p[k].grad).norm() <= room * p[k].grad.norm(), k
    # a training step as the trainers make it, and evaluation on the users x items grid
    users, pos = users[:64].to(DEV), items[:64].to(DEV)
    neg = torch.randint(0, 40, (64, 3), generator=g).to(DEV)
    opt = model.configure_optimizers()
    opt.zero_grad()
    before = {k: v.detach().clone() for k, v in model.named_parameters()}
    model.calculate_loss(((users, pos), neg)).backward()
    opt.step()
    for k, v in model.named_parameters():
        assert torch.isfinite(v).all()
        if v.requires_grad and k.startswith('combined_block'):
            assert not torch.equal(v, before[k]), k
    from collie_amd.metrics import get_preds
    model.eval()
    with torch.no_grad():
        preds = get_preds(model, torch.arange(5), 40, DEV)
        want, _ = deep_reference(model, torch.arange(5).repeat_interleave(40),
                                 torch.arange(40).repeat(5))
    assert (preds.reshape(-1).cpu().double() - want).norm() <= room * want.norm()


def _pass(F, p, call=None):
    """One block with its gradients."""
    leaves = [t.detach().requires_grad_() for t in p]
    table, norm_w, wg, wu, back, bias = leaves

    def block(table):
        h = F.embedding_rows(table, torch.arange(40, device=DEV) % table.shape[0], scale=0.5)
        g = F.gated_linear(F.layer_norm(h, norm_w), wg, wu)
        return F.linear(g, back, bias, 'gelu', residual=h)

    y = call(block, table) if call else block(table)
    return [y, *torch.autograd.grad((y * y).sum(), leaves)]


def _block_parameters():
    shapes = [(17, 24), (24,), (36, 24), (36, 24), (24, 36), (24,)]
    return [rand(s, torch.float32, 70 + i).to(DEV) for i, s in enumerate(shapes)]


def test_saved_tensors_may_be_packed_or_computed_again():
    from torch.utils.checkpoint import checkpoint

    from collie_amd import functional as F
    p = _block_parameters()
    ref = _pass(F, p)
    again = _pass(F, p, lambda block, t: checkpoint(block, t, use_reentrant=False))
    with torch.autograd.graph.save_on_cpu():
        packed = _pass(F, p)
    for other in (again, packed):
        assert all(torch.equal(a, b) for a, b in zip(ref, other))


def test_threads_on_streams_of_their_own_give_the_same():
    from concurrent.futures import ThreadPoolExecutor

    from collie_amd import functional as F
    p = _block_parameters()
    ref = _pass(F, p)
    torch.cuda.synchronize()

    def work(_):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            out = [_pass(F, p) for _ in range(5)]
        stream.synchronize()
        return out

    with ThreadPoolExecutor(4) as pool:
        for results in pool.map(work, range(4)):
            for other in results:
                assert all(torch.equal(a, b) for a, b in zip(ref, other))


def test_a_captured_block_replays_with_eager_work_between():
    from collie_amd import functional as F
    p = _block_parameters()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):
            _pass(F, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = _pass(F, p)
    for turn in range(3):
        for t in p:
            t.mul_(1.0 + 0.25 * turn)
        graph.replay()
        torch.cuda.synchronize()
        eager = _pass(F, p)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
