"""
The layers of a deeper ranking head as differentiable functions of tensors on a HIP device:
embedding rows with scaling, layer normalisation, the linear layer with bias, activation and
residual, and the gated layer.  ``collie_amd.layers`` has them as modules.

Inputs are float32, bfloat16 or float16 (all of one call alike; under ``torch.autocast`` the caller
casts); sums, statistics and activations are computed in float32 and every result of a forward pass is
rounded once.  Gradients are summed in a fixed order: equal calls give equal bits.  Layers other than
the embedding rows can be differentiated once.

Three things are not as float32 would have them.  In bfloat16 and float16 the gradient before an
activation (``dy f'(z)``; of the gated layer both) is rounded to the type before it is multiplied with
the weights and the inputs, so their gradients are 1.4 times one rounding off; in float16 a part of it
below 2^-25 is lost and one past 1.6e7 is infinite (the bias gradients are sums of the unrounded ones).
In float32, matrix products are made of bfloat16 ones, exact to float32's own rounding for magnitudes
from about 2^-110 up; smaller values keep fewer digits.

There is no CPU fallback.  What torch records or transforms by its own calls does not see these: tensors
under ``vmap``, ``torch.func`` or ``torch.jit.trace``, fake tensors and forward-mode tangents are refused
(the tables of ``collie_amd.layers``, called as modules, then do what ``torch.nn.Embedding`` does).

Everything is launched on the current stream of the inputs' device and can be captured into a graph.
As with any torch operation, drop eager results that depend on the same leaves before a backward pass
is captured: autograd would otherwise accumulate on the stream of the eager one.
"""
import torch

from collie_amd import _lib, ops


def embedding_rows(weight, ids, scale=1.0, padding_idx=None, sparse=False, status=None):
    """
    ``scale * weight[ids]``, [*ids.shape, dim].  An id outside the table gives a row of zeros, takes
    no gradient and sets bit 0 of ``status`` (int32 [1], optional).  Row ``padding_idx`` is looked up
    like any other but takes no gradient.  The gradient of ``weight`` is dense, or the uncoalesced
    COO tensor of ``nn.Embedding(sparse=True)`` with ``sparse``.
    """
    return _lib.load_autograd().embedding_rows(weight, ids, scale, padding_idx, sparse, status)


# Rows from which on a table's dense gradient is summed by sorted ids.  Below, the handful of launches
# costs more than torch's atomic adds even on skewed ids (11,264 x 128 into 138,493 rows: 63 us sorted,
# 23 us uniform and 57 us skewed with atomics, 9 us of each for the check of the ids); above, skewed ids
# meet on a few rows and the adds queue up (65,536 x 128: 70 us sorted, 51 and 264 us with atomics;
# 720,896 x 128: 164 us against 2.6 ms).
SORTED_GRAD_ROWS = 65536


def table_grad(table, ids, vals, status=None):
    """Dense gradient of ``table`` (float32) from one row of ``vals`` per id, as ``nn.Embedding``
    gives it; many rows are summed by sorted ids, in the order of the batch.  Ids outside the table
    take no gradient (the lookup has set bit 0 of ``status`` for them)."""
    rows = table.shape[0]
    vals = vals.reshape(ids.shape[0], table.shape[1])
    if not SORTED_GRAD_ROWS <= ids.shape[0] < 1 << 30:     # (the sorted form ends there)
        # index_add_ does not look at the ids on every build of torch: those outside the table (-1 and
        # `rows` after the clamp, `rows` after the remainder) go to a row behind it
        inside = ids.long().clamp(-1, rows).remainder_(rows + 1)
        return table.new_zeros(rows + 1, table.shape[1]).index_add_(0, inside, vals)[:rows]
    return ops.embedding_rows_grad(ids, vals, rows, status=status)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.  ``weight`` and
    ``bias`` ([dim], optional) are float32 or of ``x``'s type."""
    return _lib.load_autograd().layer_norm(x, weight, bias, eps)


def linear(x, weight, bias=None, activation='identity', residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one launch: ``weight`` [n_out, n_in],
    ``bias`` [n_out], ``residual`` of the result's shape; ``activation`` is 'identity', 'relu',
    'leaky_relu' (slope 0.01, as in the hybrid head), 'sigmoid', 'silu' or 'gelu' (erf)."""
    return _lib.load_autograd().linear(x, weight, bias, ops.activation_code(activation), residual)


def gated_linear(x, gate_weight, up_weight, gate_bias=None, up_bias=None, activation='silu'):
    """``activation(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)``: both products,
    the activation and the product of the two in one launch; weights [n_out, n_in], both biases or
    none; activations as for ``linear``."""
    return _lib.load_autograd().gated_linear(x, gate_weight, up_weight, gate_bias, up_bias,
                                             ops.activation_code(activation))
