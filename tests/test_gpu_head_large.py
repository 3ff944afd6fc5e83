"""
GPU tests (``-m gpu``) of the ranking-head operators on tensors of more than 2^32 values: addresses past
32 bits, on whole numbers whose sums are exact.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
M = (1 << 25) + 3                   # rows; times 136 columns: 4.56e9 values, 9.1 GB of bfloat16
WIDE = 136
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip('needs 120 GB of free memory')
    yield
    torch.cuda.empty_cache()


def signs(shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, 2, shape, generator=g, device=DEV, dtype=torch.int8).mul_(2).sub_(1).to(BF16)


def spots():
    """Row blocks at both ends and around the borders of 2^31 and 2^32 values."""
    at = [0, (1 << 31) // WIDE, (1 << 32) // WIDE, M - 200]
    return [slice(a, a + 200) for a in at]


def test_lookup_and_its_gradient():
    from collie_amd import functional as F
    table = signs((1000, WIDE), 1).requires_grad_()
    ids = torch.arange(M, device=DEV) % 1000
    y = F.embedding_rows(table, ids)
    for s in spots():
        assert torch.equal(y[s].detach(), table.detach()[ids[s]])
    dy = torch.zeros_like(y)
    for s in spots():
        dy[s] = 1.0
    (grad,) = torch.autograd.grad(y, [table], dy)
    count = torch.zeros(1000, device=DEV)
    for s in spots():
        count += torch.bincount(ids[s], minlength=1000)
    assert torch.equal(grad, count.to(BF16)[:, None].expand(1000, WIDE))


def test_layer_norm():
    from collie_amd import functional as F
    x = signs((M, WIDE), 2).requires_grad_()
    y = F.layer_norm(x)
    dy = torch.ones_like(y)
    (dx,) = torch.autograd.grad(y, [x], dy)
    for s in spots():
        part = x.detach()[s].clone().requires_grad_()
        z = F.layer_norm(part)
        assert torch.equal(y[s], z)
        assert torch.equal(dx[s], torch.autograd.grad(z, [part], dy[s])[0])


@pytest.mark.parametrize('n_in,n_out', [(WIDE, 8), (8, WIDE)])
def test_linear(n_in, n_out):
    from collie_amd import functional as F
    x, w = signs((M, n_in), 3).requires_grad_(), signs((n_out, n_in), 4).requires_grad_()
    y = F.linear(x, w, activation='relu')
    dy = torch.zeros_like(y)
    for s in spots():
        dy[s] = signs((200, n_out), s.start)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    total = torch.zeros(n_out, n_in, dtype=torch.float64, device=DEV)
    for s in spots():
        xs, w64, d = x.detach()[s].double(), w.detach().double(), dy[s].double()
        z = torch.mm(xs, w64.T.contiguous())
        assert torch.equal(y[s].detach(), z.clamp(min=0).float().to(BF16))
        dz = d * (z > 0)
        assert torch.equal(dx[s], torch.mm(dz, w64).float().to(BF16))
        total += torch.mm(dz.T.contiguous(), xs)
    assert torch.equal(dw, total.float().to(BF16))


def test_gated():
    from collie_amd import functional as F
    x, wg, wu = (signs(s, i).requires_grad_() for i, s in enumerate([(M, 8), (WIDE, 8), (WIDE, 8)]))
    y = F.gated_linear(x, wg, wu, activation='relu')
    dy = torch.zeros_like(y)
    for s in spots():
        dy[s] = signs((200, WIDE), s.start)
    dx, dwg, dwu = torch.autograd.grad(y, [x, wg, wu], dy)
    sums = [torch.zeros(WIDE, 8, dtype=torch.float64, device=DEV) for _ in range(2)]
    for s in spots():
        xs, g64, u64, d = x.detach()[s].double(), wg.detach().double(), wu.detach().double(), dy[s].double()
        g, u = torch.mm(xs, g64.T.contiguous()), torch.mm(xs, u64.T.contiguous())
        assert torch.equal(y[s].detach(), (g.clamp(min=0) * u).float().to(BF16))
        dg, du = d * u * (g > 0), d * g.clamp(min=0)
        assert torch.equal(dx[s], (torch.mm(dg, g64) + torch.mm(du, u64)).float().to(BF16))
        sums[0] += torch.mm(dg.T.contiguous(), xs)
        sums[1] += torch.mm(du.T.contiguous(), xs)
    assert torch.equal(dwg, sums[0].float().to(BF16)) and torch.equal(dwu, sums[1].float().to(BF16))
