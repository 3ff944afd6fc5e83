"""
The operators of a deeper ranking head, as cases that can be timed and compared: the embedding
lookup and its gradient by sorted ids, layer normalisation, the linear layer with bias, activation
and residual, and the gated layer.  ``own`` selects between the plain torch form (float32 whatever
the inputs' type, rounded once at the end) and this package's calls (``collie_amd.functional``).

A training case returns the output and the gradient of every input; the gradient of the output is
an input.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
LEAKY_SLOPE = 0.01

# no case, listed or drawn, goes past these
MAX_EMBED_VALUES = 1 << 26            # looked-up values, and values of the table
MAX_NORM_VALUES = 720_896 * 128
MAX_FLOPS = {'f32': 0.6e12, 'bf16': 2.2e12, 'f16': 2.2e12}     # of a whole pass
MAX_ROW_VALUES = 1.8e8                # rows x (in + out)


def listed():
    return [
        # one batch of the default size looks its users up (26,744 x 64 is the ML-20M item table)
        {'name': 'lookup-batch', 'op': 'embedding', 'dtype': 'f32', 'train': False, 'rows': 26744,
         'dim': 64, 'n': 1024, 'ids': 'uniform', 'scale': 1.0},
        # the large training batch on the ML-20M user table, skewed as real users are
        {'name': 'lookup-train-users', 'op': 'embedding', 'dtype': 'f32', 'train': True,
         'rows': 138493, 'dim': 64, 'n': 1048576, 'ids': 'zipf', 'scale': 1.0},
        # 65,536 samples with ten negatives each, on the item table, in half the bytes
        {'name': 'lookup-train-items-bf16', 'op': 'embedding', 'dtype': 'bf16', 'train': True,
         'rows': 26744, 'dim': 128, 'n': 720896, 'ids': 'zipf', 'scale': 8.0},
        # scoring one pair: nothing but latency
        {'name': 'norm-one-row', 'op': 'norm', 'dtype': 'f32', 'train': False, 'rows': 1,
         'dim': 128},
        # the hybrid head's batch (65,536 samples x 11 pairs) at its first layer's width
        {'name': 'norm-train-pairs', 'op': 'norm', 'dtype': 'f32', 'train': True, 'rows': 720896,
         'dim': 128},
        # wide rows of a width that no vector divides
        {'name': 'norm-train-odd-bf16', 'op': 'norm', 'dtype': 'bf16', 'train': True,
         'rows': 24001, 'dim': 1023},
        # scoring one pair through a wide layer: the weights are read once, for one row
        {'name': 'linear-one-row-bf16', 'op': 'linear', 'dtype': 'bf16', 'train': False, 'rows': 1,
         'n_in': 1024, 'n_out': 4096, 'bias': True, 'act': 'leaky_relu', 'residual': False},
        # the first combined layer of the hybrid head on a training batch
        {'name': 'linear-train-pairs', 'op': 'linear', 'dtype': 'f32', 'train': True,
         'rows': 720896, 'n_in': 256, 'n_out': 128, 'bias': True, 'act': 'gelu',
         'residual': False},
        # the projection back of a wide block, added to the block's input
        {'name': 'linear-train-back-bf16', 'op': 'linear', 'dtype': 'bf16', 'train': True,
         'rows': 16384, 'n_in': 5504, 'n_out': 2048, 'bias': True, 'act': 'identity',
         'residual': True},
        # a few pairs, widths that nothing divides
        {'name': 'gated-few-odd-f16', 'op': 'gated', 'dtype': 'f16', 'train': False, 'rows': 13,
         'n_in': 509, 'n_out': 1361, 'bias': True, 'act': 'silu'},
        # a block at the head's own width, in its own type
        {'name': 'gated-train-f32', 'op': 'gated', 'dtype': 'f32', 'train': True, 'rows': 65536,
         'n_in': 256, 'n_out': 512, 'bias': True, 'act': 'silu'},
        # the wide block: all matrix products
        {'name': 'gated-train-wide-bf16', 'op': 'gated', 'dtype': 'bf16', 'train': True,
         'rows': 16384, 'n_in': 2048, 'n_out': 5504, 'bias': False, 'act': 'silu'},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['embedding', 'norm', 'linear', 'gated'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    train = rng.random() < 0.7
    case = {'op': op, 'dtype': dtype, 'train': train}
    if op == 'embedding':
        dim = _spread(rng, 8, 512)
        case.update(rows=_spread(rng, 100, min(1_000_000, MAX_EMBED_VALUES // dim)), dim=dim,
                    n=_spread(rng, 16, min(1_048_576, MAX_EMBED_VALUES // dim)),
                    ids=rng.choice(['uniform', 'zipf']), scale=rng.choice([1.0, math.sqrt(dim)]))
    elif op == 'norm':
        dim = _spread(rng, 16, 8192)
        case.update(rows=_spread(rng, 1, min(720_896, MAX_NORM_VALUES // dim)), dim=dim)
    else:
        n_in, n_out = _spread(rng, 16, 4096), _spread(rng, 16, 5504)
        per_row = 2.0 * n_in * n_out * (3 if train else 1) * (2 if op == 'gated' else 1)
        most = int(min(720_896, MAX_FLOPS[dtype] / per_row, MAX_ROW_VALUES / (n_in + n_out)))
        case.update(rows=_spread(rng, 1, max(1, most)), n_in=n_in, n_out=n_out,
                    bias=rng.random() < 0.5)
        if op == 'linear':
            # the slope of relu and leaky_relu jumps at zero: among many sums a few lie so near it
            # that float32 puts them on the other side, so their gradients cannot be compared here
            smooth = ['identity', 'sigmoid', 'silu', 'gelu']
            case.update(act=rng.choice(smooth if train else smooth + ['relu', 'leaky_relu']),
                        residual=rng.random() < 0.5)
        else:
            case.update(act=rng.choice(['silu', 'gelu', 'sigmoid']))
    return case


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case['dtype']]

    def normal(*shape, std=1.0, leaf=True):
        t = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(std).to(dtype)
        return t.requires_grad_(case['train']) if leaf else t

    s = {'case': case}
    op = case['op']
    if op == 'embedding':
        rows, n = case['rows'], case['n']
        u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
        if case['ids'] == 'zipf':       # popularity ~ rank^-1.05 over a shuffled table
            e = 1.0 - 1.05
            rank = ((float(rows + 1) ** e - 1.0) * u + 1.0) ** (1.0 / e) - 1.0
            shuffle = torch.randperm(rows, generator=gen, device=dev)
            s['ids'] = shuffle[rank.long().clamp_(0, rows - 1)]
        else:
            s['ids'] = (u * rows).long().clamp_(0, rows - 1)
        s['weight'] = normal(rows, case['dim'], std=0.1)
        if case['train']:
            s['dy'] = normal(n, case['dim'], leaf=False)
    elif op == 'norm':
        rows, dim = case['rows'], case['dim']
        s['x'] = normal(rows, dim)
        s['weight'] = (1.0 + normal(dim, std=0.1, leaf=False).float()).to(dtype)
        s['weight'].requires_grad_(case['train'])
        s['bias'] = normal(dim, std=0.1)
        if case['train']:
            s['dy'] = normal(rows, dim, leaf=False)
    else:
        rows, n_in, n_out = case['rows'], case['n_in'], case['n_out']
        std = 1.0 / math.sqrt(n_in)
        s['x'] = normal(rows, n_in)
        if op == 'linear':
            s['weight'] = normal(n_out, n_in, std=std)
            s['bias'] = normal(n_out, std=0.1) if case['bias'] else None
            s['residual'] = normal(rows, n_out) if case['residual'] else None
        else:
            s['gate_weight'] = normal(n_out, n_in, std=std)
            s['up_weight'] = normal(n_out, n_in, std=std)
            s['gate_bias'] = normal(n_out, std=0.1) if case['bias'] else None
            s['up_bias'] = normal(n_out, std=0.1) if case['bias'] else None
        if case['train']:
            s['dy'] = normal(rows, n_out, leaf=False)
    return s


# the order in which a training pass returns its gradients
LEAVES = {'embedding': ('weight',), 'norm': ('x', 'weight', 'bias'),
          'linear': ('x', 'weight', 'bias', 'residual'),
          'gated': ('x', 'gate_weight', 'up_weight', 'gate_bias', 'up_bias')}


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _PLAIN[s['case']['op']](s)


def _run_own(s):
    from collie_amd import functional as F
    case = s['case']
    op = case['op']
    with torch.set_grad_enabled(case['train']):
        if op == 'embedding':
            y = F.embedding_rows(s['weight'], s['ids'], scale=case['scale'])
        elif op == 'norm':
            y = F.layer_norm(s['x'], s['weight'], s['bias'])
        elif op == 'linear':
            y = F.linear(s['x'], s['weight'], s['bias'], activation=case['act'],
                         residual=s['residual'])
        else:
            y = F.gated_linear(s['x'], s['gate_weight'], s['up_weight'], s['gate_bias'],
                               s['up_bias'], activation=case['act'])
    if not case['train']:
        return [y]
    leaves = [s[k] for k in LEAVES[op] if s[k] is not None]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s['dy']))


# ---- the plain forms ---------------------------------------------------------------------------
def _act(z, kind):
    """(act(z), act'(z))"""
    if kind == 'identity':
        return z, torch.ones_like(z)
    if kind == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if kind == 'leaky_relu':
        slope = torch.where(z > 0, torch.ones_like(z), torch.full_like(z, LEAKY_SLOPE))
        return z * slope, slope
    if kind == 'gelu':
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-z))
    if kind == 'sigmoid':
        return sig, sig * (1.0 - sig)
    return z * sig, sig * (1.0 + z * (1.0 - sig))       # silu


def _plain_embedding(s):
    case, w, ids = s['case'], s['weight'], s['ids']
    out = [(w.float()[ids] * case['scale']).to(w.dtype)]
    if case['train']:
        grad = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        grad.index_add_(0, ids, s['dy'].float() * case['scale'])
        out.append(grad.to(w.dtype))
    return out


def _plain_norm(s, eps=1e-5):
    dtype = s['x'].dtype
    x, w, b = s['x'].float(), s['weight'].float(), s['bias'].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + eps)
    xhat = xc * rstd
    out = [(xhat * w + b).to(dtype)]
    if s['case']['train']:
        dy = s['dy'].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        out += [dx.to(dtype), (dy * xhat).sum(0).to(dtype), dy.sum(0).to(dtype)]
    return out


def _plain_linear(s):
    case, dtype = s['case'], s['x'].dtype
    x, w = s['x'].float(), s['weight'].float()
    z = x @ w.t()
    if s['bias'] is not None:
        z = z + s['bias'].float()
    a, da = _act(z, case['act'])
    y = a + s['residual'].float() if s['residual'] is not None else a
    out = [y.to(dtype)]
    if case['train']:
        dz = s['dy'].float() * da
        out += [(dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
        if s['bias'] is not None:
            out.append(dz.sum(0).to(dtype))
        if s['residual'] is not None:
            out.append(s['dy'].clone())
    return out


def _plain_gated(s):
    case, dtype = s['case'], s['x'].dtype
    x, wg, wu = s['x'].float(), s['gate_weight'].float(), s['up_weight'].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s['gate_bias'] is not None:
        g, u = g + s['gate_bias'].float(), u + s['up_bias'].float()
    a, da = _act(g, case['act'])
    out = [(a * u).to(dtype)]
    if case['train']:
        dy = s['dy'].float()
        dg, du = dy * u * da, dy * a
        out += [(dg @ wg + du @ wu).to(dtype), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype)]
        if s['gate_bias'] is not None:
            out += [dg.sum(0).to(dtype), du.sum(0).to(dtype)]
    return out


_PLAIN = {'embedding': _plain_embedding, 'norm': _plain_norm, 'linear': _plain_linear,
          'gated': _plain_gated}


# ---- the definition in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    """Each operator's definition in float64; gradients by torch's differentiation of it."""
    s = prepare(case, seed)
    op = case['op']
    t = {k: v.detach().double() for k, v in s.items()
         if torch.is_tensor(v) and v.is_floating_point()}
    leaves = [t[k].requires_grad_(case['train']) for k in LEAVES[op] if s[k] is not None]

    def activation(z):
        return {'identity': lambda: z, 'relu': lambda: z.clamp(min=0.0),
                'leaky_relu': lambda: torch.maximum(z, z * LEAKY_SLOPE),
                'sigmoid': lambda: torch.sigmoid(z), 'silu': lambda: z * torch.sigmoid(z),
                'gelu': lambda: z * torch.special.ndtr(z)}[case['act']]()

    def affine(weight, bias):
        z = torch.mm(t['x'], t[weight].T.contiguous())
        return z if bias not in t else z + t[bias]

    with torch.set_grad_enabled(case['train']):
        if op == 'embedding':
            y = t['weight'].index_select(0, s['ids']) * case['scale']
        elif op == 'norm':
            var, mean = torch.var_mean(t['x'], dim=1, correction=0, keepdim=True)
            y = (t['x'] - mean) * (var + 1e-5).rsqrt() * t['weight'] + t['bias']
        elif op == 'linear':
            y = activation(affine('weight', 'bias'))
            if 'residual' in t:
                y = y + t['residual']
        else:
            y = activation(affine('gate_weight', 'gate_bias')) * affine('up_weight', 'up_bias')
    if not case['train']:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, t['dy']))


def work(case):
    size = 4 if case['dtype'] == 'f32' else 2
    op, train = case['op'], case['train']
    if op == 'embedding':
        rows, dim, n = case['rows'], case['dim'], case['n']
        found = min(rows, n)        # rows of the table that can be looked up at all
        data = (n + found) * dim * size + 8 * n
        flops = n * dim
        if train:
            data += (n + rows) * dim * size
            flops += n * dim
        return {'bytes': data, 'flops': flops}
    if op == 'norm':
        values = case['rows'] * case['dim']
        return {'bytes': size * ((4 if train else 2) * values + (4 if train else 2) * case['dim']),
                'flops': (19 if train else 8) * values}
    rows, n_in, n_out = case['rows'], case['n_in'], case['n_out']
    pair = 2 if op == 'gated' else 1
    weights = pair * n_in * n_out + (pair * n_out if case['bias'] else 0)
    values = rows * (n_in + n_out) + weights
    flops = 2 * pair * rows * n_in * n_out
    if train:       # dy in; dx and the weights' gradients out
        values += rows * (n_in + n_out) + weights
        flops *= 3
    if case.get('residual'):
        values += (2 if train else 1) * rows * n_out
    return {'bytes': size * values, 'flops': flops}
