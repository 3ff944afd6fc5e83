"""
The ranking-head operators in float64 and, for each result, a bound on the error of a computation
that sums in float32, keeps what the backward pass needs in the inputs' type and rounds the result
once.  ``U[t]`` is half a step of type t, F = U[float32]; a float32 sum of n terms is off by at most
n F times the sum of their magnitudes.
"""
import math

import torch

F = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# smallest normal number / 2 steps: results below it are rounded absolutely
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def check(got, want, bound, dtype):
    """|got - want| <= bound + one rounding, element by element."""
    assert got.dtype == dtype and got.shape == want.shape, (got.dtype, got.shape, want.shape)
    if want.numel() == 0:
        return
    got = got.double().cpu()
    # a value past the type's largest number is infinite: it must be where all of [want - bound,
    # want + bound] is past it, and may be where some of it is
    most = torch.finfo(dtype).max
    inf = torch.isinf(got) & (want.abs() + bound > most) & (got.sign() * want + bound > most)
    assert inf[want.abs() - bound > most].all()
    err = torch.where(inf, torch.zeros_like(want), (got - want).abs())
    room = bound + U[dtype] * (want.abs() + bound) + TINY[dtype]
    worst = (err / room).max().item()
    assert torch.isfinite(err).all() and worst <= 1.0, f'error is {worst:.3g} of its bound'


def act(z, kind):
    """f, f', a bound on |f'| and a bound on |f''| away from the kinks."""
    if kind == 'identity':
        return z, torch.ones_like(z), 1.0, 0.0
    if kind == 'relu':
        return z.clamp(min=0), (z > 0).double(), 1.0, 0.0
    if kind == 'leaky_relu':
        s = torch.where(z > 0, 1.0, 0.01).double()
        return z * s, s, 1.0, 0.0
    if kind == 'sigmoid':
        s = torch.sigmoid(z)
        return s, s * (1 - s), 0.25, 0.1
    if kind == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 1.1, 0.5
    cdf = torch.special.ndtr(z)
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13, 0.8


def product(a, b, b_err=0.0, a_err=0.0):
    """a @ b.T and the bound of its float32 sum (operands off by a_err / b_err)."""
    n = a.shape[1]
    mag = a.abs() @ b.abs().T
    err = (n + 2) * F * mag
    if not isinstance(a_err, float):
        err = err + a_err @ b.abs().T * (1 + (n + 2) * F)
    if not isinstance(b_err, float):
        err = err + a.abs() @ b_err.T
    return a @ b.T, err


def _affine(x, w, bias):
    z, ez = product(x, w)
    if bias is not None:
        z = z + bias
        ez = ez + F * (z.abs() + ez)
    return z, ez


def _kept(z, ez, kind, dtype):
    """(f, f', errors of both) computed from z as it is kept."""
    f, d, l1, l2 = act(z, kind)
    err = ez + U[dtype] * (z.abs() + ez) + TINY[dtype]
    ef = l1 * err + 16 * F * (z.abs() + 1)
    ed = l2 * err + 16 * F * (z.abs() + 1)
    if kind in ('relu', 'leaky_relu'):      # on either side of the kink
        ed = torch.where(z.abs() <= err, torch.ones_like(ed), ed)
    return f, d, ef, ed


def linear(x, w, bias, residual, kind, dy, dtype):
    """{name: (value, bound)} for y, dx, dw, db of the linear layer, from float64 tensors."""
    z, ez = _affine(x, w, bias)
    f, d, l1, _ = act(z, kind)
    ey = l1 * ez + 16 * F * (z.abs() + 1)
    y = f
    if residual is not None:
        y = f + residual
        ey = ey + F * (y.abs() + ey)
    out = {'y': (y, ey)}
    if dy is None:
        return out
    if kind == 'identity':
        dz, e = dy, torch.zeros_like(dy)
    else:
        _, d, _, ed = _kept(z, ez, kind, dtype)
        dz = dy * d
        e = dy.abs() * ed + 2 * F * dz.abs()
    out['db'] = (dz.sum(0), e.sum(0) + (len(dz) + 20) * F * dz.abs().sum(0))
    e = e + U[dtype] * (dz.abs() + e) + TINY[dtype]     # dz is kept in the inputs' type
    out['dx'] = product(dz, w.T, a_err=e)
    out['dw'] = product(dz.T, x.T, a_err=e.T)
    return out


def gated(x, wg, wu, bg, bu, kind, dy, dtype):
    g, eg = _affine(x, wg, bg)
    u, eu = _affine(x, wu, bu)
    f, _, l1, _ = act(g, kind)
    ef = l1 * eg + 16 * F * (g.abs() + 1)
    y = f * u
    out = {'y': (y, ef * (u.abs() + eu) + f.abs() * eu + F * y.abs())}
    if dy is None:
        return out
    f, d, ef, ed = _kept(g, eg, kind, dtype)
    eu = eu + U[dtype] * (u.abs() + eu) + TINY[dtype]
    dg, du = dy * u * d, dy * f
    edg = dy.abs() * (eu * (d.abs() + ed) + u.abs() * ed) + 4 * F * dg.abs()
    edu = dy.abs() * ef + 2 * F * du.abs()
    for name, v, e in (('dbg', dg, edg), ('dbu', du, edu)):
        out[name] = (v.sum(0), e.sum(0) + (len(v) + 20) * F * v.abs().sum(0))
    edg = edg + U[dtype] * (dg.abs() + edg) + TINY[dtype]
    edu = edu + U[dtype] * (du.abs() + edu) + TINY[dtype]
    out['dx'] = product(torch.cat([dg, du], 1), torch.cat([wg, wu]).T,
                        a_err=torch.cat([edg, edu], 1))
    out['dwg'] = product(dg.T, x.T, a_err=edg.T)
    out['dwu'] = product(du.T, x.T, a_err=edu.T)
    return out


def layer_norm(x, w, b, eps, dy, dtype):
    """Values a lane adds one by one, then a tree over at most 256 lanes."""
    D = x.shape[1]
    chain = (min(D, 64) if D <= 8192 else D // 256 + 8) + 12
    c = chain * F
    m = x.mean(1, keepdim=True)
    em = c * x.abs().mean(1, keepdim=True)
    xc = x - m
    v = (xc * xc).mean(1, keepdim=True)
    exc = em + F * xc.abs()
    # (xc + e)^2 = xc^2 + 2 e xc + e^2
    ev = (2 * xc.abs() * exc + exc * exc).mean(1, keepdim=True) + (c + 4 * F) * v
    r = (v + eps).rsqrt()
    er = ev / (2 * (v + eps)) + 4 * F       # relative; first order, and ev is far below v + eps
    h = xc * r
    eh = (exc + xc.abs() * (er + 2 * F)) * r * 1.01
    y = h * w + b
    out = {'y': (y, w.abs() * eh + 2 * F * ((h * w).abs() + b.abs()))}
    if dy is None:
        return out
    g = dy * w
    eg = F * g.abs()
    m1, m2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    e1 = (c + 2 * F) * g.abs().mean(1, keepdim=True)
    e2 = (g.abs() * eh).mean(1, keepdim=True) + (c + 4 * F) * (g * h).abs().mean(1, keepdim=True)
    inner = g - m1 - h * m2
    ei = (eg + e1 + h.abs() * e2 + eh * (m2.abs() + e2)
          + 4 * F * (g.abs() + m1.abs() + (h * m2).abs()))
    out['dx'] = (r * inner, r * (ei + (er + 2 * F) * (inner.abs() + ei)) * 1.01)
    n = len(x) + 20
    out['dw'] = ((dy * h).sum(0), (dy.abs() * eh).sum(0) + n * F * (dy * h).abs().sum(0))
    out['db'] = (dy.sum(0), n * F * dy.abs().sum(0))
    return out
