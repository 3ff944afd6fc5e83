"""
GPU tests (``-m gpu``) of the linear and gated layers over every tile of the matrix kernels, whole and cut
along the depth (``head_tiles``).  Inputs are small whole numbers: every product, sum and activation is
exact in float32 whatever the order, so results have to be those of float64 rounded once, bit for bit.
"""
import pytest
import torch

import head_bounds as hb
import head_tiles as ht

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
CASES = [(t, *c) for t in (torch.bfloat16, torch.float16) for c in ht.SIXTEEN_BITS]
CASES += [(torch.float32, *c) for c in ht.FLOAT32]


def signs(gen, shape, density):
    """-1, 0 and 1, not 0 with the given probability."""
    s = torch.randint(0, 2, shape, generator=gen, device=DEV, dtype=torch.float32).mul_(2).sub_(1)
    return s.mul_(torch.rand(shape, generator=gen, device=DEV) < density)


def relu_slope(z):
    return (z > 0).double()


@pytest.mark.parametrize('dtype,gated,m,n_in,n_out', CASES)
def test_every_tile_exactly(dtype, gated, m, n_in, n_out):
    from collie_amd import functional as F
    gen = torch.Generator(device=DEV).manual_seed(m + 3 * n_in + 7 * n_out)
    # sums have a variance of at most 600, so that |u| stays below 256 and every dg, du is a number of
    # all three types; sums of n_out or m of them stay below 2^24
    x = signs(gen, (m, n_in), min(0.7, 900.0 / n_in))
    w, dy = signs(gen, (n_out, n_in), 0.6), signs(gen, (m, n_out), 0.7)
    b = torch.randint(-3, 4, (n_out,), generator=gen, device=DEV).float()
    more = signs(gen, (n_out, n_in), 0.6) if gated else signs(gen, (m, n_out), 0.7)
    b2 = torch.randint(-3, 4, (n_out,), generator=gen, device=DEV).float()
    leaves = [t.to(dtype).requires_grad_() for t in ((x, w, more, b, b2) if gated else (x, w, b, more))]
    if gated:
        y = F.gated_linear(*leaves, activation='relu')
    else:
        y = F.linear(*leaves[:3], activation='relu', residual=leaves[3])
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy.to(dtype))]

    x, w, dy, b, b2, more = (t.double() for t in (x, w, dy, b, b2, more))
    z = torch.mm(x, w.T.contiguous()) + b
    if gated:
        u = torch.mm(x, more.T.contiguous()) + b2
        assert z.abs().max() <= 256 and u.abs().max() <= 256
        dg, du = dy * u * relu_slope(z), dy * z.clamp(min=0)
        want = [z.clamp(min=0) * u, torch.mm(dg, w) + torch.mm(du, more),
                torch.mm(dg.T.contiguous(), x), torch.mm(du.T.contiguous(), x), dg.sum(0), du.sum(0)]
    else:
        dz = dy * relu_slope(z)
        want = [z.clamp(min=0) + more, torch.mm(dz, w), torch.mm(dz.T.contiguous(), x), dz.sum(0), dy]
    for i, (g, v) in enumerate(zip(got, want)):
        assert v.abs().max() < 2 ** 24
        assert torch.equal(g, v.float().to(dtype)), i


@pytest.mark.parametrize('m,n_in,n_out', [c[1:] for c in ht.FLOAT32 if not c[0]])
def test_float32_tiles_with_all_digits(m, n_in, n_out):
    """The parts that float32 values are split into, in every tile."""
    from collie_amd import functional as F
    gen = torch.Generator(device=DEV).manual_seed(m + n_in)
    x, w, dy = (torch.randn(s, generator=gen, device=DEV) for s in ((m, n_in), (n_out, n_in), (m, n_out)))
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    y = F.linear(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    x, w, dy = x.double(), w.double(), dy.double()
    for g, (a, b) in zip(got, ((x, w.T.contiguous()), (dy, w), (dy.T.contiguous(), x))):
        # hb.product's bound, made on the device
        room = (a.shape[1] + 2) * hb.F * torch.mm(a.abs(), b.abs())
        want = torch.mm(a, b)
        assert ((g.double() - want).abs() <= room + hb.F * want.abs()).all()
