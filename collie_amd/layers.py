"""
Parameter containers of the MF model (reference: ``collie/model/base/layers.py``).

The tables are ``torch.nn.Embedding`` subclasses, so that ``state_dict()`` keys, shapes, the
``sparse`` flag and the initial distributions are those of the reference.  The fused paths look rows
up inside their own kernels, straight from ``.weight``; a table that is called as a module takes
``functional.embedding_rows`` on a HIP device, where an id outside the table gives a row of zeros and
an ``IndexError`` at the next ``check_status()``.

``LayerNorm``, ``Linear`` and ``GatedLinear`` are the layers of a deeper ranking head
(``collie_amd.functional``) with the parameter names and the initialisation of their ``torch.nn``
counterparts.
"""
from typing import Dict, List, Optional

import torch

from collie_amd import _lib, functional


class Table(torch.nn.Embedding):
    # int32 [1] on the table's device once it has been called there: bit 0 says that an id was outside
    _status = None

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if torch.jit.is_scripting():        # (the other branch is not compiled then)
            return torch.nn.functional.embedding(
                input, self.weight, self.padding_idx, self.max_norm, self.norm_type,
                self.scale_grad_by_freq, self.sparse)
        else:
            if not self._kernels_take(input):
                return super().forward(input)
            return functional.embedding_rows(self.weight, input, padding_idx=self.padding_idx,
                                             sparse=self.sparse, status=self._status_flag())

    @torch.jit.unused
    def _status_flag(self):
        if self._status is None or self._status.device != self.weight.device:
            if torch.cuda.is_current_stream_capturing():
                return None     # memory of the graph, which would clear it with every replay
            with torch.inference_mode(False):       # (check_status writes to it outside of that mode)
                self._status = torch.zeros(1, dtype=torch.int32, device=self.weight.device)
        return self._status

    @torch.jit.unused
    def check_status(self):
        """Raise ``IndexError`` if a call since the last check had an id outside the table (syncs).
        On a HIP device such an id gives a row of zeros and takes no gradient; the models look here
        where they look at the flag of their own kernels (``MatrixFactorizationModel.check_status``)."""
        if self._status is not None and int(self._status.item()) & 1:
            self._status.zero_()
            raise IndexError('index out of range in self: an id is outside the table')

    @torch.jit.unused
    def _kernels_take(self, input) -> bool:
        # What the kernels do not take stays torch's: other devices and types, empty tables and those
        # past the entry points' limits, renormalised rows, gradients divided by counts; and calls that
        # stand for others (recorded, compiled or transformed ones, tensors with forward-mode tangents).
        if (torch.compiler.is_compiling() or torch.jit.is_tracing()
                or torch.overrides.has_torch_function((input, self.weight))):
            return False
        return (self.weight.is_cuda and self.weight.numel() > 0
                and self.weight.shape[0] < (1 << 31) - 1 and self.weight.shape[1] <= 1 << 20
                and input.numel() < 1 << 30
                and self.weight.dtype in _lib.ELEMENT_TYPES
                and input.is_cuda and input.dtype in (torch.int32, torch.int64)
                and self.max_norm is None and not self.scale_grad_by_freq
                and _lib.load_autograd().plain(self.weight)
                and _lib.load_autograd().plain(input))


class ScaledEmbedding(Table):
    """N(0, (1 / (2.5 * embedding_dim))^2) initialisation (``layers.py:6-10``)."""

    def reset_parameters(self) -> None:
        self.weight.data.normal_(0, 1.0 / (self.embedding_dim * 2.5))


class ZeroEmbedding(Table):
    """All-zero initialisation (``layers.py:13-17``)."""

    def reset_parameters(self) -> None:
        self.weight.data.zero_()


class LayerNorm(torch.nn.LayerNorm):
    """``torch.nn.LayerNorm`` over the last dimension (``functional.layer_norm``)."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None):
        if not isinstance(normalized_shape, int):
            raise ValueError('LayerNorm normalises the last dimension only: expected an int, not '
                             f'{normalized_shape!r}')
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if input.shape[-1:] != self.normalized_shape:
            raise ValueError(f'expected [..., {self.normalized_shape[0]}], not {tuple(input.shape)}')
        return functional.layer_norm(input, self.weight, self.bias, self.eps)


class Linear(torch.nn.Linear):
    """``torch.nn.Linear`` with an activation and an optional residual that is added to its result
    (``functional.linear``)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: str = 'identity', device=None, dtype=None):
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f'{activation!r} is not an activation: {", ".join(_lib.ACTIVATIONS)}')
        super().__init__(in_features, out_features, bias, device, dtype)
        self.activation = activation

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return functional.linear(input, self.weight, self.bias, self.activation, residual)


class GatedLinear(torch.nn.Module):
    """``activation(gate(x)) * up(x)`` with two ``torch.nn.Linear`` parameter sets ``gate`` and
    ``up`` (``functional.gated_linear``)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: str = 'silu', device=None, dtype=None):
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f'{activation!r} is not an activation: {", ".join(_lib.ACTIVATIONS)}')
        super().__init__()
        self.gate = torch.nn.Linear(in_features, out_features, bias, device, dtype)
        self.up = torch.nn.Linear(in_features, out_features, bias, device, dtype)
        self.activation = activation

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return functional.gated_linear(input, self.gate.weight, self.up.weight, self.gate.bias,
                                       self.up.bias, self.activation)


class MultiOptimizer(object):
    """``zero_grad`` over a list of optimizers (``layers.py:20-38``)."""

    def __init__(self, optimizers: List[torch.optim.Optimizer]):
        assert isinstance(optimizers, list), f'Expected list, got {type(optimizers)}!'
        self.optimizers = optimizers

    def zero_grad(self) -> None:
        for optimizer in self.optimizers:
            optimizer.zero_grad()


class MultiLRScheduler(object):
    """``step`` over a list of ``{'scheduler': ...}`` dicts (``layers.py:41-63``)."""

    def __init__(self, lr_schedulers: List[Dict[str, object]]):
        assert isinstance(lr_schedulers, list), f'Expected list, got {type(lr_schedulers)}!'
        self.lr_schedulers = [d['scheduler'] for d in lr_schedulers]

    def step(self, *args, **kwargs) -> None:
        for lr_scheduler in self.lr_schedulers:
            lr_scheduler.step(*args, **kwargs)
