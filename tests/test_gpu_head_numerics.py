"""
GPU tests (``-m gpu``) of the ranking-head operators where their numbers are hard: large constants under
a layer norm, tails of activations, and intermediate values at the ends of a type's range.
"""
import pytest
import torch

import head_bounds as hb

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
TYPES = [torch.float32, torch.bfloat16, torch.float16]
F = hb.F


# ---- layer norm of rows that lie far from zero -----------------------------------------------------
def chain(dim):
    """Roundings of a sum over a row: values that one lane adds, then a tree (see hb.layer_norm)."""
    return (min(dim, 64) if dim <= 8192 else dim // 256 + 8) + 12


DIMS = [7, 30, 109, 255, 600, 1023, 3001, 8193, 20011]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', DIMS)
def test_layer_norm_of_large_constant_rows(dim, dtype):
    """The mean c (1 + d) is off by |d| <= chain F, what is left of a value, c d, is exact, and so is its
    mean but for chain + 2 roundings: at most c chain (chain + 2) F^2 stays, over sqrt(eps)."""
    from collie_amd import functional
    c = {torch.float32: 1e6, torch.bfloat16: 999424.0, torch.float16: 60000.0}[dtype]
    x = torch.tensor([c, -c, c / 4]).to(dtype)[:, None].expand(3, dim).contiguous()
    leaf = x.to(DEV).requires_grad_()
    y = functional.layer_norm(leaf)
    k = chain(dim)
    assert y.detach().abs().max().item() <= c * k * (k + 2) * F * F / 1e-5 ** 0.5
    # the gradient of a row without variance is (dy - mean(dy)) / sqrt(eps): its inner product with the
    # row's values, all alike, is part of what is rounded
    dy = torch.ones_like(y)
    (dx,) = torch.autograd.grad(y, [leaf], dy)
    assert dx.abs().max().item() <= 4 * k * F / 1e-5 ** 0.5


@pytest.mark.parametrize('dim', DIMS)
def test_layer_norm_of_rows_with_a_large_mean(dim):
    """Whole numbers around 1e6: differences from the mean of their first rounding are exact, so the
    result and its gradients keep float32's accuracy relative to the largest of the row."""
    from collie_amd import functional
    g = torch.Generator().manual_seed(dim)
    x = 1e6 + torch.randint(-3, 4, (5, dim), generator=g).float()
    w, dy = torch.randn(dim, generator=g), torch.randn(5, dim, generator=g)
    leaves = [x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()]
    y = functional.layer_norm(*leaves)
    dx, dw = torch.autograd.grad(y, leaves, dy.to(DEV))
    x, w, dy = x.double(), w.double(), dy.double()
    xc = x - x.mean(1, keepdim=True)
    var = (xc * xc).mean(1, keepdim=True)
    r = (var + 1e-5).rsqrt()
    h = xc * r
    k = chain(dim)
    # relative error of rstd: half of what k + 6 roundings do to the squares, which contain the square of
    # the first mean's error (k F 1e6 at most) until that is taken out again
    er = (k + 6) * F * (1 + (k * F * 1e6) ** 2 / var)
    # (v - off): off is off by k + 2 roundings of the mean of |v|, v by nothing
    eh = (k + 8) * F * (h.abs().mean(1, keepdim=True) + h.abs()) + h.abs() * er
    room = eh * w.abs() + 2 * F * (h * w).abs() + F * (h * w).abs()
    hb.check(y.detach(), h * w, room, torch.float32)
    gr = dy * w
    m1, m2 = gr.mean(1, keepdim=True), (gr * h).mean(1, keepdim=True)
    e1 = (k + 4) * F * gr.abs().mean(1, keepdim=True)
    e2 = (gr.abs() * eh).mean(1, keepdim=True) + (k + 6) * F * (gr * h).abs().mean(1, keepdim=True)
    inner = gr - m1 - h * m2
    ei = F * gr.abs() + e1 + h.abs() * e2 + eh * (m2.abs() + e2) + 4 * F * (gr.abs() + m1.abs()
                                                                             + (h * m2).abs())
    hb.check(dx, r * inner, r * (ei + (er + 2 * F) * (inner.abs() + ei)) * 1.01, torch.float32)
    hb.check(dw, (dy * h).sum(0), (dy.abs() * eh).sum(0) + 25 * F * (dy * h).abs().sum(0), torch.float32)


# ---- activations far from zero ---------------------------------------------------------------------
def test_gelu_keeps_the_digits_of_its_tail():
    """z Phi(z) and its slope in float32, one column, weight one.  Phi: the exponential and its two parts
    (4 F with the instruction), the polynomial (its own 1 F, 4 F of rounding), the reciprocal (2 F, which
    t times the polynomial feels at most twice), three products; with the product by z 16 F at most."""
    from collie_amd import functional
    z = torch.cat([torch.linspace(-12.4, 9.0, 30001), torch.tensor([0.0, -0.0, 1e-30, -1e-30])])
    z = z.reshape(-1, 1)
    x, w = z.to(DEV).requires_grad_(), torch.ones(1, 1, device=DEV)
    y = functional.linear(x, w, activation='gelu')
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    z = z.double()
    phi, pdf = torch.special.log_ndtr(z).exp(), torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    tiny = 2.0 ** -126                      # (z = 1e-30 is kept, its square is not)
    assert ((y.double().cpu() - z * phi).abs() <= 16 * F * (z * phi).abs() + tiny).all()
    # Phi + z pdf(z): both to 16 F, their sum, dz and the product (four dropped parts) round once each
    room = 20 * F * (phi + (z * pdf).abs()) + tiny
    assert ((dx.double().cpu() - (phi + z * pdf)).abs() <= room).all()


@pytest.mark.parametrize('dtype', TYPES[1:])
@pytest.mark.parametrize('kind', ['sigmoid', 'silu', 'gelu'])
def test_slopes_are_those_of_the_unrounded_sums(kind, dtype):
    """z = a + b with b far below a's last bits, so z has more digits than the inputs' type.  dz is rounded
    to that type and dx = dz is not again: one half step of the slope, and what float32 leaves of it (F of
    the terms whose sum it is, 20 of them at most, sigmoid's 1 - s being F e^|z| off)."""
    from collie_amd import functional
    a = torch.linspace(-9, 9, 4001).to(dtype)
    b = (a.float().abs() * hb.U[dtype] * torch.rand(4001, generator=torch.Generator().manual_seed(1)))
    x = torch.stack([a, b.to(dtype)], 1)
    leaf, w = x.to(DEV).requires_grad_(), torch.ones(1, 2, dtype=dtype, device=DEV)
    y = functional.linear(leaf, w, activation=kind)
    (dx,) = torch.autograd.grad(y, [leaf], torch.ones_like(y))
    z = x.double().sum(1)
    _, slope, _, _ = hb.act(z, kind)
    terms = 20 * F * (1 + z.abs()) if kind != 'sigmoid' else 20 * F * torch.sigmoid(z)
    room = hb.U[dtype] * slope.abs() + terms + hb.TINY[dtype]
    for col in range(2):
        err = (dx[:, col].double().cpu() - slope).abs()
        assert (err <= room).all(), (err / room).max()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ['relu', 'leaky_relu'])
def test_slope_of_sums_below_the_range_of_the_type(kind, dtype):
    """x w is positive and rounds to zero in float16: the slope is that of the positive side."""
    from collie_amd import functional
    small = {torch.float32: 2.0 ** -60, torch.bfloat16: 2.0 ** -60, torch.float16: 2.0 ** -14}[dtype]
    x = torch.tensor([[small], [-small], [0.0]], dtype=dtype, device=DEV).requires_grad_()
    w = torch.full((1, 1), small, dtype=dtype, device=DEV)
    y = functional.linear(x, w, activation=kind)
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    low = 0.0 if kind == 'relu' else torch.tensor(0.01).to(dtype).item() * small
    want = torch.tensor([[small], [low], [low]]).to(dtype)
    assert torch.equal(dx.cpu(), want)


# ---- float16: activation gradients past the type's range -------------------------------------------
def gated_case(m, n_in, n_out, seed):
    """Ordinary values, and in some rows |dy u f'(g)| up to 5e5 where the weights are small."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n_in, generator=g) * 0.25
    wg = torch.randn(n_out, n_in, generator=g) / 64
    wu = torch.randn(n_out, n_in, generator=g) / 64
    bg, bu = torch.randn(n_out, generator=g), torch.randn(n_out, generator=g)
    dy = torch.randn(m, n_out, generator=g)
    bu[0], dy[m // 2, 0], dy[-1, 0] = 700.0, 600.0, -600.0
    return [t.half() for t in (x, wg, wu, bg, bu, dy)]


def check_gated(kind, case, run):
    x, wg, wu, bg, bu, dy = case
    ref = hb.gated(*(t.double() for t in (x, wg, wu, bg, bu)), kind, dy.double(), torch.float16)
    assert (dy.double() * (x.double() @ wu.double().T + bu.double())).abs().max() > 4e5
    names = ('dx', 'dwg', 'dwu', 'dbg', 'dbu')
    # stored times 1 / 256, a value is off by half of 2^-24 times 256, wherever it is
    low = 2.0 ** -17
    more = {'dx': low * (wg.double().abs().sum(0) + wu.double().abs().sum(0)).expand(len(x), -1),
            'dwg': low * x.double().abs().sum(0).expand(len(wg), -1)}
    more['dwu'] = more['dwg']
    for name, g in zip(names, run):
        val, bound = ref[name]
        hb.check(g, val, bound + more.get(name, 0.0), torch.float16)
    # (hb.check lets a value be infinite only where the exact one may round to that: 4.2e5 |x| in dwg's
    # first row does for |x| > 0.156)
    assert torch.isfinite(run[0]).all()


OVER = [(2, 24, 40), (70, 33, 130), (5000, 64, 48), (300, 520, 264)]


@pytest.mark.parametrize('kind', ['identity', 'silu', 'leaky_relu'])
@pytest.mark.parametrize('m,n_in,n_out', OVER)
def test_float16_gated_gradients_past_the_range(m, n_in, n_out, kind):
    from collie_amd import functional
    case = gated_case(m, n_in, n_out, m)
    leaves = [t.to(DEV).requires_grad_() for t in case[:5]]
    y = functional.gated_linear(*leaves, activation=kind)
    grads = torch.autograd.grad(y, leaves, case[5].to(DEV), retain_graph=True)
    check_gated(kind, case, grads)
    # a call in range afterwards is what it was before: nothing is kept
    small = (case[5] / 1024).to(DEV)
    first = torch.autograd.grad(y, leaves, small, retain_graph=True)
    again = torch.autograd.grad(y, leaves, case[5].to(DEV), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, small)))


@pytest.mark.parametrize('kind', ['silu', 'gelu'])
def test_float16_linear_gradients_past_the_range(kind):
    """The slopes of silu and gelu go past one."""
    from collie_amd import functional
    x = torch.tensor([[2.0, 0.5], [1.4, 0.25]]).half()
    w, dy = torch.tensor([[1.0, 1 / 64]]).half() / 2, torch.tensor([[65000.0], [-65000.0]]).half()
    x[:, 0] = 2.4 * 2 if kind == 'silu' else 1.4 * 2
    leaves = [x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()]
    y = functional.linear(*leaves, activation=kind)
    dx, dw = torch.autograd.grad(y, leaves, dy.to(DEV))
    ref = hb.linear(x.double(), w.double(), None, None, kind, dy.double(), torch.float16)
    assert (dy.double() * hb.act(x.double() @ w.double().T, kind)[1]).abs().min() > 65600
    hb.check(dx, *ref['dx'], torch.float16)
    hb.check(dw, *ref['dw'], torch.float16)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_float16_gradients_past_the_range_in_a_captured_pass():
    from collie_amd import functional
    case = gated_case(70, 33, 130, 3)
    leaves = [t.to(DEV).requires_grad_() for t in case[:5]]
    dy = case[5].to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(functional.gated_linear(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(functional.gated_linear(*leaves), leaves, dy)
    for factor in (1 / 1024, 1.0, 1 / 1024, 1.0):       # in range and past it, in turn
        dy.copy_((case[5].float() * factor).half().to(DEV))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        eager = torch.autograd.grad(functional.gated_linear(*leaves), leaves, dy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        if factor == 1.0:
            check_gated('silu', case, got)


# ---- how far 16-bit gradients are, in the mean -----------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES[1:])
@pytest.mark.parametrize('gated', [False, True])
def test_gradients_are_two_roundings_off_in_the_mean(gated, dtype):
    """dz (dg, du) is rounded to the type, and so is the result: two independent errors of one size, 1.41
    times one of them in the 2-norm.  Keeping the gated layer's pre-activations in 16 bits too would give
    1.8.  60,000 values: the ratio is known to one percent."""
    from collie_amd import functional
    g = torch.Generator().manual_seed(5)
    m, n_in, n_out = 200, 300, 128
    x = torch.randn(m, n_in, generator=g).to(dtype)
    w, w2 = ((torch.randn(n_out, n_in, generator=g) * n_in ** -0.5).to(dtype) for _ in range(2))
    dy = torch.randn(m, n_out, generator=g).to(dtype)
    leaves = [t.to(DEV).requires_grad_() for t in ((x, w, w2) if gated else (x, w))]
    y = (functional.gated_linear(*leaves) if gated else functional.linear(*leaves, activation='silu'))
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    ref = (hb.gated(x.double(), w.double(), w2.double(), None, None, 'silu', dy.double(), dtype) if gated
           else hb.linear(x.double(), w.double(), None, None, 'silu', dy.double(), dtype))
    for name, grad in zip(('dx', 'dwg', 'dwu') if gated else ('dx', 'dw'), got):
        want = ref[name][0]
        one = (want.to(dtype).double() - want).norm()
        ratio = ((grad.cpu().double() - want).norm() / one).item()
        print(name, ratio)
        assert ratio < 1.6, (name, ratio)


def test_float32_products_of_small_values():
    """A value is split into three bfloat16 parts, the last a multiple of 2^-133: off by half of that, and by
    nothing from 2^-110 on (24 bits reach 2^-133).  One column, weights powers of two: no other rounding
    but that of results below 2^-126."""
    from collie_amd import functional
    g = torch.Generator().manual_seed(2)
    e = torch.arange(-126, -60).repeat_interleave(8)
    x = torch.ldexp(1 + torch.rand(len(e), generator=g), e)[:, None]
    for power in (0, 20):
        y = functional.linear(x.to(DEV), torch.full((70, 1), 2.0 ** power, device=DEV)).cpu().double()
        want = x.double() * 2.0 ** power
        lost = torch.where(e[:, None] < -110, 2.0 ** -134, 0.0).double() * 2.0 ** power
        assert ((y - want).abs() <= lost).all()
