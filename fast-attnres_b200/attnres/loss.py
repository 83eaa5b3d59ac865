"""Language-model head and loss in one operator, without the logits.

The last read of a network goes through a bias-free head ``[V, D]`` into a softmax cross entropy
(benchmarks/model.py:336-338 and benchmarks/training_graph.py:24-58 of the reference).  As separate
operations that keeps ``[N, V]`` logits, their FP32 copy and their gradient (5 GB for 16 384
positions of a 32 000-word vocabulary); here the logits exist one tile at a time.

    loss = linear_cross_entropy(last_read, lm_head.weight, targets)
    # == F.cross_entropy((last_read @ lm_head.weight.T).float(), targets)
"""
from __future__ import annotations

import math

import torch

from . import _calls, _native
from ._sources import MAX_WIDTH, _first_failure, check_scalar

# Compiled operators (csrc/torch_ops.cpp): `linear_cross_entropy_forward` and `..._backward`, or
# `..._with_gradients` and `..._scale_gradient`, launch the kernels; `linear_cross_entropy` is the
# differentiable call over either pair.
_ops = _native.load_operators()
_linear_cross_entropy = _ops.linear_cross_entropy.default
_TYPES = _calls.HALVES
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MAX_ROWS = 1 << 30


def _loss_like(hidden, targets, reduction):
    return hidden.new_empty(targets.shape if reduction == 0 else (), dtype=torch.float32)


@torch.library.register_fake("attnres_b200::linear_cross_entropy_forward")
def _(hidden, weight, targets, ignored, reduction, scale):
    width = hidden.shape[-1]
    rows = hidden.numel() // width
    return (_loss_like(hidden, targets, reduction),
            hidden.new_empty((rows, (width + 7) // 8 * 8)),
            hidden.new_empty((2, rows), dtype=torch.int32),
            hidden.new_empty((1,), dtype=torch.int32),
            hidden.new_empty((rows,), dtype=torch.float32))


@torch.library.register_fake("attnres_b200::linear_cross_entropy_backward")
def _(grad, weight, targets, kept, index, count, sums, ignored, reduction, scale, need_hidden,
      need_weight):
    return (weight.new_empty((*targets.shape, weight.shape[1]) if need_hidden else (0,)),
            weight.new_empty(weight.shape if need_weight else (0,)))


@torch.library.register_fake("attnres_b200::linear_cross_entropy_with_gradients")
def _(hidden, weight, targets, ignored, reduction, scale, need_hidden, need_weight):
    return (_loss_like(hidden, targets, reduction),
            hidden.new_empty(hidden.shape if need_hidden else (0,)),
            hidden.new_empty(weight.shape if need_weight else (0,)))


@torch.library.register_fake("attnres_b200::linear_cross_entropy_scale_gradient")
def _(gradient, upstream):
    return torch.empty_like(gradient, memory_format=torch.contiguous_format)


@torch.library.register_fake("attnres_b200::linear_cross_entropy")
def _(hidden, weight, targets, ignored, reduction, scale):
    return _loss_like(hidden, targets, reduction)


def _check(hidden, weight, targets, ignore_index, reduction, scale) -> None:
    _first_failure((
        (lambda: all(isinstance(t, torch.Tensor) for t in (hidden, weight, targets)), TypeError,
         "hidden, weight and targets must be tensors"),
        (lambda: hidden.dtype in _TYPES, TypeError, "hidden must be BF16 or FP16"),
        (lambda: weight.dtype == hidden.dtype, TypeError, "weight must have hidden's type"),
        (lambda: targets.dtype in (torch.int64, torch.int32), TypeError,
         "targets must be int64 or int32"),
        (lambda: weight.device == hidden.device and targets.device == hidden.device, TypeError,
         "hidden, weight and targets must be on one device"),
        (lambda: hidden.ndim >= 1 and 1 <= hidden.shape[-1] <= MAX_WIDTH, ValueError,
         f"expected hidden [...,D] with 1<=D<={MAX_WIDTH}"),
        (lambda: weight.ndim == 2 and weight.shape[1] == hidden.shape[-1], ValueError,
         "weight must have shape [V,D]"),
        (lambda: 1 <= weight.shape[0] <= _calls.MAX_VOCABULARY, ValueError,
         f"supported vocabulary is 1<=V<={_calls.MAX_VOCABULARY}"),
        (lambda: targets.shape == hidden.shape[:-1], ValueError,
         "targets must have hidden's leading axes"),
        (lambda: targets.numel() <= MAX_ROWS, ValueError, "too many rows"),
        (lambda: reduction in _REDUCTIONS, ValueError,
         "reduction must be 'mean', 'sum' or 'none'"),
        (lambda: isinstance(ignore_index, int) and not isinstance(ignore_index, bool), TypeError,
         "ignore_index must be an integer"),
    ))
    check_scalar(scale, "scale")
    if not hidden.is_cuda:
        raise RuntimeError("linear_cross_entropy requires CUDA tensors")


def _acceptable(hidden, weight, targets) -> bool:
    """The conditions of `_check` on the tensors at the cost of a call on a few rows; `_check`
    names the one that does not hold."""
    return (isinstance(hidden, torch.Tensor) and isinstance(weight, torch.Tensor)
            and isinstance(targets, torch.Tensor) and hidden.is_cuda and hidden.dtype in _TYPES
            and weight.dtype == hidden.dtype and targets.dtype in _calls.INTEGERS
            and weight.device == hidden.device and targets.device == hidden.device
            and hidden.ndim > 0 and 1 <= hidden.shape[-1] <= MAX_WIDTH and weight.ndim == 2
            and weight.shape[1] == hidden.shape[-1]
            and 1 <= weight.shape[0] <= _calls.MAX_VOCABULARY
            and targets.shape == hidden.shape[:-1] and targets.numel() <= MAX_ROWS)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean",
                         scale: float = 1.0) -> torch.Tensor:
    """``F.cross_entropy(scale * hidden @ weight.T, targets)`` in FP32, logits never kept.

    ``hidden``: ``[..., D]``, ``weight``: ``[V, D]``, both BF16 or both FP16; ``targets``: int64 or
    int32 ids of ``hidden``'s leading shape.  Rows whose target is ``ignore_index`` take no part:
    they cost no products, their loss and gradient are zero whatever they hold.  Any other target
    outside the vocabulary makes the loss, and the gradients, NaN.  ``reduction``: ``"mean"`` over
    the rows that count (NaN when there is none), ``"sum"``, or ``"none"`` (the shape of
    ``targets``).  The loss is FP32; products run on the tensor cores with FP32 accumulators, and
    the softmax residue is rounded to the inputs' type before it is multiplied into the gradients,
    which come back in that type.  Differentiable once; results are the same bits every time.

    A BF16 mean or sum over rows of 512 features and more forms its gradients in the forward, from
    the same logits (so evaluate under ``torch.no_grad()``); the backward multiplies them by the
    upstream gradient, one more rounding unless that is a power of two.  Every other call forms the
    logits a second time in the backward.
    """
    if not (_acceptable(hidden, weight, targets) and type(ignore_index) is int
            and reduction in _REDUCTIONS and _calls.plain_number(scale) and math.isfinite(scale)):
        _check(hidden, weight, targets, ignore_index, reduction, scale)
    return _linear_cross_entropy(hidden, weight, targets, ignore_index, _REDUCTIONS[reduction], scale)


__all__ = ["linear_cross_entropy"]
