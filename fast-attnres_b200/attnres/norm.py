"""LayerNorm over the last axis, for the places of a network that no read precedes.

In a network of reads every sublayer's norm but the first follows a read and can run in its
epilogue (``attnres.fused.attnres_layer_norm``); the first sublayer consumes the embedding itself
(benchmarks/model.py:293-311 of the reference), and a stream that is normalised without being read
needs the norm alone.

    y = layer_norm(x, norm.weight, norm.bias, norm.eps)
    # == F.layer_norm(x.float(), (D,), weight.float(), bias.float(), eps), rounded to x's type

One pass over the data forward, one backward; the parameter gradients are summed in a fixed order.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _calls, _native, _ops
from ._sources import MAX_WIDTH, _first_failure, check_scalar

_TYPES = _calls.TYPE_CODES


def _forward(x, weight, bias, eps, need_stats):
    width = x.shape[-1]
    rows = x.numel() // width
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty((2, rows if need_stats else 0), device=x.device, dtype=torch.float32)
    if rows == 0:
        return y, stats
    kept, row_stride = _calls.rows_of(x)
    parameter = weight if weight is not None else bias
    with _calls.on_device(x.device):
        _native.norm_forward(
            kept.data_ptr(), row_stride, _calls.pointer(weight), _calls.pointer(bias), rows, width,
            _TYPES[x.dtype], _TYPES[torch.float32 if parameter is None else parameter.dtype], eps,
            y.data_ptr(), stats.data_ptr() if need_stats else None, _calls.stream(x.device))
    return y, stats


def _backward(grad, x, stats, weight, param_dtype, need_x, need_weight, need_bias):
    """-> (dx, dweight, dbias), None where not needed."""
    width = x.shape[-1]
    rows = x.numel() // width
    device = x.device
    dx = torch.empty(x.shape, device=device, dtype=x.dtype) if need_x else None
    make = torch.empty if rows else torch.zeros
    dweight = make((width,), device=device, dtype=param_dtype) if need_weight else None
    dbias = make((width,), device=device, dtype=param_dtype) if need_bias else None
    if rows == 0 or not (need_x or need_weight or need_bias):
        return dx, dweight, dbias
    kept, row_stride = _calls.rows_of(x)
    upstream, grad_stride = _calls.rows_of(grad)
    with _calls.on_device(device):
        partials, partial_rows = None, 0
        if need_weight or need_bias:
            partial_rows = _native.norm_workspace_rows(rows, width, device.index)
            partials = torch.empty((partial_rows, 2 * width), device=device, dtype=torch.float32)
        _native.norm_backward(
            upstream.data_ptr(), grad_stride, kept.data_ptr(), row_stride, stats.data_ptr(),
            _calls.pointer(weight), rows, width, _TYPES[x.dtype], _TYPES[param_dtype],
            _calls.pointer(dx), _calls.pointer(partials), partial_rows, _calls.pointer(dweight),
            _calls.pointer(dbias), _calls.stream(device))
    return dx, dweight, dbias


@_ops._custom_op("attnres_b200::norm_forward", mutates_args=(), device_types="cuda")
def norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                 eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (y, stats [2, rows]: mean, 1 / standard deviation)."""
    return _forward(x, weight, bias, eps, True)


@norm_forward.register_fake
def _(x, weight, bias, eps):
    return (x.new_empty(x.shape),
            x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32))


@_ops._custom_op("attnres_b200::norm_backward", mutates_args=(), device_types="cuda")
def norm_backward(grad: torch.Tensor, x: torch.Tensor, stats: torch.Tensor,
                  weight: Optional[torch.Tensor], param_dtype: torch.dtype, need_x: bool,
                  need_weight: bool, need_bias: bool
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A gradient that is not needed comes back with 0 elements."""
    dx, dweight, dbias = _backward(grad, x, stats, weight, param_dtype, need_x, need_weight,
                                   need_bias)
    return (x.new_empty((0,)) if dx is None else dx,
            x.new_empty((0,), dtype=param_dtype) if dweight is None else dweight,
            x.new_empty((0,), dtype=param_dtype) if dbias is None else dbias)


@norm_backward.register_fake
def _(grad, x, stats, weight, param_dtype, need_x, need_weight, need_bias):
    width = x.shape[-1]
    return (x.new_empty(x.shape if need_x else (0,)),
            x.new_empty((width if need_weight else 0,), dtype=param_dtype),
            x.new_empty((width if need_bias else 0,), dtype=param_dtype))


def _param_dtype(weight, bias):
    return (weight if weight is not None else bias).dtype if (
        weight is not None or bias is not None) else torch.float32


def _op_setup(ctx, inputs, output) -> None:
    x, weight, bias, _eps = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, output[1])
    ctx.param_dtype = _param_dtype(weight, bias)


def _op_backward(ctx, grad, _grad_stats):
    if grad is None:
        return None, None, None, None
    x, weight, stats = ctx.saved_tensors
    need = [bool(n) for n in ctx.needs_input_grad[:3]]
    grads = norm_backward(grad, x, stats, weight, ctx.param_dtype, *need)
    return (*(g if n else None for g, n in zip(grads, need)), None)


torch.library.register_autograd(norm_forward, _op_backward, setup_context=_op_setup)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param_dtype = _param_dtype(weight, bias)
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return None, None, None, None
        x, weight, stats = ctx.saved_tensors
        return (*_backward(grad, x, stats, weight, ctx.param_dtype, *ctx.needs_input_grad[:3]), None)


def _check(x, weight, bias, eps) -> None:
    _first_failure((
        (lambda: isinstance(x, torch.Tensor), TypeError, "x must be a tensor"),
        (lambda: x.dtype in _TYPES, TypeError, "x must be BF16, FP16 or FP32"),
        (lambda: x.ndim >= 1 and 1 <= x.shape[-1] <= MAX_WIDTH, ValueError,
         f"expected x [...,D] with 1<=D<={MAX_WIDTH}"),
    ))
    for name, parameter in (("weight", weight), ("bias", bias)):
        if parameter is None:
            continue
        _first_failure((
            (lambda: isinstance(parameter, torch.Tensor), TypeError, f"{name} must be a tensor"),
            (lambda: parameter.dtype in _TYPES, TypeError, f"{name} must be BF16, FP16 or FP32"),
            (lambda: parameter.device == x.device, TypeError, f"{name} must be on x's device"),
            (lambda: parameter.shape == (x.shape[-1],), ValueError, f"{name} must have shape [D]"),
        ))
    check_scalar(eps, "eps")
    if eps < 0:
        raise ValueError("eps must not be negative")
    if not x.is_cuda:
        raise RuntimeError("layer_norm requires CUDA tensors")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, in ``x``'s type.

    ``x``: ``[..., D]`` in BF16, FP16 or FP32, ``1 <= D <= 8192``, any strides (rows that one
    stride cannot walk, or whose features are apart, are copied first).  ``weight`` / ``bias``:
    ``[D]`` in any of the three types (used in FP32, their gradients come back in their own type),
    or None for ones / zeros.  Mean, variance and every sum are FP32; the result is rounded once.
    Differentiable once; no row at all gives an empty result and zero parameter gradients.
    """
    _check(x, weight, bias, eps)
    if weight is not None:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
        if weight is not None and bias.dtype != weight.dtype:
            # one type for both inside the kernel; FP32 holds the other two exactly
            weight, bias = weight.float(), bias.float()
    eps = float(eps)
    if not _calls.direct(x, weight, bias):
        return norm_forward(x, weight, bias, eps)[0]
    if _calls.wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


__all__ = ["layer_norm"]
