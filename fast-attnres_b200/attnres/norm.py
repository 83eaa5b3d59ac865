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

import math

import torch

from . import _calls, _native
from ._sources import MAX_WIDTH, _first_failure, check_scalar

# The work is done by torch operators compiled from csrc/torch_ops.cpp: `norm_forward` and
# `norm_backward` launch the kernels, `layer_norm` is the differentiable call over the two.
_ops = _native.load_operators()
_layer_norm = _ops.layer_norm.default
_TYPES = _calls.FLOATS


@torch.library.register_fake("attnres_b200::norm_forward")
def _(x, weight, bias, eps, need_stats):
    rows = x.numel() // x.shape[-1] if need_stats else 0
    return x.new_empty(x.shape), x.new_empty((2, rows), dtype=torch.float32)


@torch.library.register_fake("attnres_b200::norm_backward")
def _(grad, x, stats, weight, param_type, need_x, need_weight, need_bias):
    width = x.shape[-1]
    return (x.new_empty(x.shape if need_x else (0,)),
            x.new_empty((width if need_weight else 0,), dtype=param_type),
            x.new_empty((width if need_bias else 0,), dtype=param_type))


@torch.library.register_fake("attnres_b200::layer_norm")
def _(x, weight, bias, eps):
    return x.new_empty(x.shape)


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


def _parameter_ok(parameter, x) -> bool:
    return (isinstance(parameter, torch.Tensor) and parameter.dtype in _TYPES
            and parameter.device == x.device and parameter.shape == x.shape[-1:])


def _acceptable(x, weight) -> bool:
    """The conditions of `_check` at the cost of a call on a few rows; `_check` names the one that
    does not hold."""
    return (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in _TYPES and x.ndim > 0
            and 1 <= x.shape[-1] <= MAX_WIDTH and (weight is None or _parameter_ok(weight, x)))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, in ``x``'s type.

    ``x``: ``[..., D]`` in BF16, FP16 or FP32, ``1 <= D <= 8192``, any strides (rows that one
    stride cannot walk, or whose features are apart, are copied first).  ``weight`` / ``bias``:
    ``[D]`` in any of the three types (used in FP32, their gradients come back in their own type),
    or None for ones / zeros.  Mean, variance and every sum are FP32; the result is rounded once.
    Differentiable once; no row at all gives an empty result and zero parameter gradients.
    """
    if not (_acceptable(x, weight) and (bias is None or _parameter_ok(bias, x))
            and _calls.plain_number(eps) and 0.0 <= eps < math.inf):
        _check(x, weight, bias, eps)
    if weight is not None:
        if not weight.is_contiguous():
            weight = weight.contiguous()
        if bias is not None and bias.dtype != weight.dtype:
            # one type for both inside the kernel; FP32 holds the other two exactly
            weight, bias = weight.float(), bias.float()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return _layer_norm(x, weight, bias, eps)


__all__ = ["layer_norm"]
