"""Language-model head and loss in one operator, without the logits.

The last read of a network goes through a bias-free head ``[V, D]`` into a softmax cross entropy
(benchmarks/model.py:336-338 and benchmarks/training_graph.py:24-58 of the reference).  As separate
operations that keeps ``[N, V]`` logits, their FP32 copy and their gradient (5 GB for 16 384
positions of a 32 000-word vocabulary); here the logits exist one tile at a time.

    loss = linear_cross_entropy(last_read, lm_head.weight, targets)
    # == F.cross_entropy((last_read @ lm_head.weight.T).float(), targets)
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _calls, _native, _ops
from ._sources import MAX_WIDTH, _first_failure, check_scalar

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MAX_ROWS = 1 << 30


def _forward(hidden, weight, targets, ignore_index, reduction, scale):
    """-> (loss, kept rows, their indices, their targets, their count, log2 of their sums)."""
    width, vocabulary, device = hidden.shape[-1], weight.shape[0], hidden.device
    rows = hidden.numel() // width
    kept = torch.empty((rows, (width + 7) // 8 * 8), device=device, dtype=hidden.dtype)
    index = torch.empty((2, rows), device=device, dtype=torch.int32)
    count = torch.empty((1,), device=device, dtype=torch.int32)
    sums = torch.empty((2, rows), device=device, dtype=torch.float32)
    loss = sums[1] if reduction == 0 else torch.empty((), device=device, dtype=torch.float32)
    if rows == 0:
        count.zero_()
        if reduction != 0:
            loss.fill_(0.0 if reduction == 1 else float("nan"))
        return loss.reshape(targets.shape) if reduction == 0 else loss, kept, index, count, sums[0]
    source, row_stride = _calls.rows_of(hidden)
    head, head_stride = _calls.rows_of(weight)
    ids = targets.contiguous()
    with _calls.on_device(device):
        size = _native.loss_workspace_bytes(rows, vocabulary, width, False)
        workspace = torch.empty((size,), device=device, dtype=torch.uint8)
        _native.loss_forward(
            source.data_ptr(), row_stride, head.data_ptr(), head_stride, ids.data_ptr(),
            ids.dtype == torch.int64, rows, vocabulary, width, _TYPES[hidden.dtype], ignore_index,
            scale, reduction, kept.data_ptr(), index.data_ptr(), index.data_ptr() + 4 * rows,
            count.data_ptr(), sums.data_ptr(), sums.data_ptr() + 4 * rows, loss.data_ptr(),
            workspace.data_ptr(), size, _calls.stream(device))
    return loss.reshape(targets.shape) if reduction == 0 else loss, kept, index, count, sums[0]


def _backward(grad, weight, targets, kept, index, count, sums, shape, ignore_index, reduction,
              scale, need_hidden, need_weight):
    """-> (dhidden, dweight), None where not needed."""
    width, vocabulary, device = weight.shape[1], weight.shape[0], weight.device
    rows = targets.numel()
    dhidden = torch.empty(shape, device=device, dtype=weight.dtype) if need_hidden else None
    make = torch.empty if rows else torch.zeros
    dweight = make((vocabulary, width), device=device, dtype=weight.dtype) if need_weight else None
    if rows == 0 or not (need_hidden or need_weight):
        return dhidden, dweight
    head, head_stride = _calls.rows_of(weight)
    ids = targets.contiguous()
    upstream = grad.reshape(-1) if grad.is_contiguous() else grad.contiguous().reshape(-1)
    with _calls.on_device(device):
        size = _native.loss_workspace_bytes(rows, vocabulary, width, True)
        workspace = torch.empty((size,), device=device, dtype=torch.uint8)
        _native.loss_backward(
            upstream.data_ptr(), 1, head.data_ptr(), head_stride, ids.data_ptr(),
            ids.dtype == torch.int64, rows, vocabulary, width, _TYPES[weight.dtype], ignore_index,
            scale, reduction, kept.data_ptr(), index.data_ptr(), index.data_ptr() + 4 * rows,
            count.data_ptr(), sums.data_ptr(), _calls.pointer(dhidden), _calls.pointer(dweight),
            workspace.data_ptr(), size, _calls.stream(device))
    return dhidden, dweight


@_ops._custom_op("attnres_b200::linear_cross_entropy_forward", mutates_args=(), device_types="cuda")
def linear_cross_entropy_forward(
        hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int,
        reduction: int, scale: float
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (loss, kept rows, [indices, targets] of the kept rows, their count, log2 of their sums)."""
    loss, kept, index, count, sums = _forward(hidden, weight, targets, ignore_index, reduction, scale)
    if reduction == 0:
        loss = loss.clone()   # outputs of an operator do not share storage
    return loss, kept, index, count, sums.clone()


@linear_cross_entropy_forward.register_fake
def _(hidden, weight, targets, ignore_index, reduction, scale):
    width = hidden.shape[-1]
    rows = hidden.numel() // width
    return (hidden.new_empty(targets.shape if reduction == 0 else (), dtype=torch.float32),
            hidden.new_empty((rows, (width + 7) // 8 * 8)),
            hidden.new_empty((2, rows), dtype=torch.int32),
            hidden.new_empty((1,), dtype=torch.int32),
            hidden.new_empty((rows,), dtype=torch.float32))


@_ops._custom_op("attnres_b200::linear_cross_entropy_backward", mutates_args=(),
                 device_types="cuda")
def linear_cross_entropy_backward(
        grad: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, kept: torch.Tensor,
        index: torch.Tensor, count: torch.Tensor, sums: torch.Tensor, ignore_index: int,
        reduction: int, scale: float, need_hidden: bool, need_weight: bool
) -> tuple[torch.Tensor, torch.Tensor]:
    """A gradient that is not needed comes back with 0 elements."""
    dhidden, dweight = _backward(grad, weight, targets, kept, index, count, sums,
                                 (*targets.shape, weight.shape[1]), ignore_index, reduction, scale,
                                 need_hidden, need_weight)
    return (weight.new_empty((0,)) if dhidden is None else dhidden,
            weight.new_empty((0,)) if dweight is None else dweight)


@linear_cross_entropy_backward.register_fake
def _(grad, weight, targets, kept, index, count, sums, ignore_index, reduction, scale, need_hidden,
      need_weight):
    return (weight.new_empty((*targets.shape, weight.shape[1]) if need_hidden else (0,)),
            weight.new_empty(weight.shape if need_weight else (0,)))


def _op_setup(ctx, inputs, output) -> None:
    _hidden, weight, targets, *ctx.constants = inputs
    ctx.mark_non_differentiable(*output[1:])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(weight, targets, *output[1:])


def _op_backward(ctx, grad, *_unused):
    if grad is None:
        return (None,) * 6
    need = bool(ctx.needs_input_grad[0]), bool(ctx.needs_input_grad[1])
    grads = linear_cross_entropy_backward(grad, *ctx.saved_tensors, *ctx.constants, *need)
    return (*(g if n else None for g, n in zip(grads, need)), None, None, None, None)


torch.library.register_autograd(linear_cross_entropy_forward, _op_backward, setup_context=_op_setup)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, *constants):
        loss, *kept = _forward(hidden, weight, targets, *constants)
        ctx.save_for_backward(weight, targets, *kept)
        ctx.set_materialize_grads(False)
        ctx.constants, ctx.shape = constants, hidden.shape
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 6
        grads = _backward(grad, *ctx.saved_tensors, ctx.shape, *ctx.constants,
                          *ctx.needs_input_grad[:2])
        return (*grads, None, None, None, None)


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
    """
    _check(hidden, weight, targets, ignore_index, reduction, scale)
    constants = ignore_index, _REDUCTIONS[reduction], float(scale)
    if not _calls.direct(hidden, weight, targets):
        return linear_cross_entropy_forward(hidden, weight, targets, *constants)[0]
    if _calls.wants_grad(hidden, weight):
        return _LinearCrossEntropy.apply(hidden, weight, targets, *constants)
    return _forward(hidden, weight, targets, *constants)[0]


__all__ = ["linear_cross_entropy"]
