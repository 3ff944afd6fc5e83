"""
The layers of a deeper ranking head as differentiable functions of tensors on a HIP device:
embedding rows with scaling, layer normalisation, the linear layer with bias, activation and
residual, and the gated layer.  ``collie_amd.layers`` has them as modules.

Inputs are float32, bfloat16 or float16 (all of one call alike; under ``torch.autocast`` the caller
casts); sums, statistics and activations are computed in float32 and every result is rounded once.
Gradients are summed in a fixed order: equal calls give equal bits.  Layers other than the embedding
rows can be differentiated once.  There is no CPU fallback.

Everything is launched on the current stream of the inputs' device and can be captured into a graph.
As with any torch operation, drop eager results that depend on the same leaves before a backward pass
is captured: autograd would otherwise accumulate on the stream of the eager one.
"""
import torch
from torch.autograd.function import once_differentiable

from collie_amd import _lib, ops


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _backward_once(fn):
    """``once_differentiable``, whose bookkeeping is left out where no second derivative can be asked
    for (without ``create_graph``: a small batch's backward pass is host time)."""
    checked = once_differentiable(fn)

    def backward(ctx, dy):
        return (checked if torch.is_grad_enabled() else fn)(ctx, dy)
    return staticmethod(backward)


class _EmbeddingRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, sparse, status):
        ctx.save_for_backward(ids)
        ctx.rest = (weight.shape, scale, padding_idx, sparse, status)
        return ops.embedding_rows(weight, ids, scale, status)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        shape, scale, padding_idx, sparse, status = ctx.rest
        if sparse:
            # the uncoalesced COO gradient of nn.Embedding(sparse=True)
            flat, vals = ids.reshape(-1).long(), dy.reshape(-1, shape[1])
            if scale != 1.0:
                vals = vals * scale
            if padding_idx is not None:
                live = flat != padding_idx
                flat, vals = flat[live], vals[live]
            return torch.sparse_coo_tensor(flat.reshape(1, -1), vals, shape), *[None] * 5
        if torch.is_grad_enabled():         # create_graph: the gradient is differentiated again
            dw = _EmbeddingRowsGrad.apply(dy, ids, shape[0], scale, padding_idx, status)
        else:
            dw = ops.embedding_rows_grad(ids, dy, shape[0], scale, padding_idx, status)
        return dw, None, None, None, None, None


class _EmbeddingRowsGrad(torch.autograd.Function):
    """The gradient is linear in ``dy``: its own gradient is the lookup again."""

    @staticmethod
    def forward(ctx, dy, ids, num_rows, scale, padding_idx, status):
        ctx.save_for_backward(ids)
        ctx.rest = (scale, padding_idx, status)
        return ops.embedding_rows_grad(ids, dy, num_rows, scale, padding_idx, status)

    @staticmethod
    def backward(ctx, ddw):
        (ids,) = ctx.saved_tensors
        scale, padding_idx, status = ctx.rest
        out = _EmbeddingRows.apply(ddw, ids, scale, padding_idx, False, status)
        if padding_idx is not None:
            out = out.masked_fill((ids == padding_idx).unsqueeze(-1), 0.0)
        return out, *[None] * 5


def embedding_rows(weight, ids, scale=1.0, padding_idx=None, sparse=False, status=None):
    """
    ``scale * weight[ids]``, [*ids.shape, dim].  An id outside the table gives a row of zeros, takes
    no gradient and sets bit 0 of ``status`` (int32 [1], optional).  Row ``padding_idx`` is looked up
    like any other but takes no gradient.  The gradient of ``weight`` is dense, or the uncoalesced
    COO tensor of ``nn.Embedding(sparse=True)`` with ``sparse``.
    """
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f'padding_idx {padding_idx} is no row of the table')
    if status is not None and (status.dtype != torch.int32 or status.device != weight.device):
        raise _lib.CollieHipError('status must be an int32 tensor on the device of the table')
    if not _wants_grad(weight):
        return ops.embedding_rows(weight, ids, scale, status)
    return _EmbeddingRows.apply(weight, ids, float(scale), padding_idx, bool(sparse), status)


# Rows from which on a table's dense gradient is summed by sorted ids.  Below, the handful of launches
# costs more than torch's atomic adds even on skewed ids (11,264 x 128 into 138,493 rows: 63 us sorted,
# 19 us uniform and 53 us skewed with atomics); above, skewed ids meet on a few rows and the adds queue
# up (65,536 x 128: 71 us sorted, 43 and 251 us with atomics; 720,896 x 128: 164 us against 2.6 ms).
SORTED_GRAD_ROWS = 65536


def table_grad(table, ids, vals, status=None):
    """Dense gradient of ``table`` (float32) from one row of ``vals`` per id, as ``nn.Embedding``
    gives it; many rows are summed by sorted ids, in the order of the batch."""
    vals = vals.reshape(ids.shape[0], table.shape[1])
    if ids.shape[0] < SORTED_GRAD_ROWS:
        return torch.zeros_like(table).index_add_(0, ids.long(), vals)
    return ops.embedding_rows_grad(ids, vals, table.shape[0], status=status)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ops.layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @_backward_once
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        return *ops.layer_norm_backward(dy, x, weight, bias, stats, ctx.needs_input_grad[:3]), None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.  ``weight`` and
    ``bias`` ([dim], optional) are float32 or of ``x``'s type."""
    if eps < 0:
        raise ValueError(f'eps must not be negative, not {eps}')
    if not _wants_grad(x, weight, bias):
        return ops.layer_norm_forward(x, weight, bias, eps, False)[0]
    return _LayerNorm.apply(x, weight, bias, eps)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        y, kept = ops.linear_forward(x, weight, bias, activation, residual,
                                     any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, kept)
        ctx.activation = activation
        return y

    @_backward_once
    def backward(ctx, dy):
        x, weight, kept = ctx.saved_tensors
        dx = dw = db = None
        if any(ctx.needs_input_grad[:3]):
            dx, dw, db = ops.linear_backward(dy, x, weight, ctx.activation, kept,
                                             ctx.needs_input_grad[:3])
        return dx, dw, db, None, dy if ctx.needs_input_grad[4] else None


def linear(x, weight, bias=None, activation='identity', residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one launch: ``weight`` [n_out, n_in],
    ``bias`` [n_out], ``residual`` of the result's shape; ``activation`` is 'identity', 'relu',
    'leaky_relu' (slope 0.01, as in the hybrid head), 'sigmoid', 'silu' or 'gelu' (erf)."""
    if not _wants_grad(x, weight, bias, residual):
        return ops.linear_forward(x, weight, bias, activation, residual, False)[0]
    return _Linear.apply(x, weight, bias, activation, residual)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, activation):
        y, gate, up = ops.gated_forward(x, gate_weight, up_weight, gate_bias, up_bias, activation,
                                        True)
        ctx.save_for_backward(x, gate_weight, up_weight, gate, up)
        ctx.activation = activation
        return y

    @_backward_once
    def backward(ctx, dy):
        x, gate_weight, up_weight, gate, up = ctx.saved_tensors
        return *ops.gated_backward(dy, x, gate_weight, up_weight, ctx.activation, gate, up,
                                   ctx.needs_input_grad[:5]), None


def gated_linear(x, gate_weight, up_weight, gate_bias=None, up_bias=None, activation='silu'):
    """``activation(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)``: both products,
    the activation and the product of the two in one launch; weights [n_out, n_in], both biases or
    none; activations as for ``linear``."""
    if not _wants_grad(x, gate_weight, up_weight, gate_bias, up_bias):
        return ops.gated_forward(x, gate_weight, up_weight, gate_bias, up_bias, activation,
                                 False)[0]
    return _Gated.apply(x, gate_weight, up_weight, gate_bias, up_bias, activation)
