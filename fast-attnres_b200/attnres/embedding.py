"""Embedding lookup with scaling and learned positions: the first source of a network of reads.

The reference's model adds a token row and a position row and casts the sum to the working type of
the stream (benchmarks/model.py:239-245 of the reference): three passes over ``[N, D]``, and a
table gradient that is scattered with atomics.  Here the lookup, the scale, the positions and the
cast are one pass, and the gradient of the table is a sum over the tokens sorted by id, in a fixed
order, so it is the same bits every time.

    first = embed(tokens, table, positions[:tokens.shape[-1]], dtype=torch.bfloat16)
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _calls, _native, _ops
from ._sources import MAX_WIDTH, _first_failure, check_scalar

_TYPES = _calls.TYPE_CODES
MAX_TOKENS = 2**31 - 1


def _period(tokens) -> int:
    return int(tokens.shape[-1]) if tokens.ndim else 1


def _forward(tokens, table, positions, scale, dtype):
    width = table.shape[1]
    out = torch.empty((*tokens.shape, width), device=table.device, dtype=dtype)
    if tokens.numel() == 0:
        return out
    ids = tokens.contiguous()
    rows, row_stride = _calls.rows_of(table)
    added, added_stride = (None, 0) if positions is None else _calls.rows_of(positions)
    with _calls.on_device(table.device):
        _native.embedding_forward(
            ids.data_ptr(), ids.dtype == torch.int64, ids.numel(), _period(ids), table.shape[0],
            width, rows.data_ptr(), row_stride, _TYPES[table.dtype], _calls.pointer(added),
            added_stride, _TYPES[torch.float32 if positions is None else positions.dtype], scale,
            out.data_ptr(), _TYPES[dtype], _calls.stream(table.device))
    return out


def _backward(grad, tokens, vocabulary, table_dtype, position_dtype, scale, padding, need_table,
              need_positions):
    """-> (dtable, dpositions), None where not needed."""
    width, device = grad.shape[-1], grad.device
    count, period = tokens.numel(), _period(tokens)
    make = torch.empty if count else torch.zeros
    dtable = make((vocabulary, width), device=device, dtype=table_dtype) if need_table else None
    dpositions = make((period, width), device=device, dtype=position_dtype) if need_positions else None
    if count == 0 or not (need_table or need_positions):
        return dtable, dpositions
    ids = tokens.contiguous()
    upstream, grad_stride = _calls.rows_of(grad)
    with _calls.on_device(device):
        workspace, size = None, 0
        if need_table:
            size = _native.embedding_workspace_bytes(count, width)
            workspace = torch.empty((size,), device=device, dtype=torch.uint8)
        _native.embedding_backward(
            ids.data_ptr(), ids.dtype == torch.int64, count, period, vocabulary, width, padding,
            upstream.data_ptr(), grad_stride, _TYPES[grad.dtype], scale, _calls.pointer(dtable),
            _TYPES[table_dtype], _calls.pointer(dpositions), _TYPES[position_dtype],
            _calls.pointer(workspace), size, _calls.stream(device))
    return dtable, dpositions


@_ops._custom_op("attnres_b200::embedding_forward", mutates_args=(), device_types="cuda")
def embedding_forward(tokens: torch.Tensor, table: torch.Tensor, positions: Optional[torch.Tensor],
                      scale: float, padding: int, dtype: torch.dtype) -> torch.Tensor:
    """`padding` (-1: none) only matters to the gradient."""
    return _forward(tokens, table, positions, scale, dtype)


@embedding_forward.register_fake
def _(tokens, table, positions, scale, padding, dtype):
    return table.new_empty((*tokens.shape, table.shape[1]), dtype=dtype)


@_ops._custom_op("attnres_b200::embedding_backward", mutates_args=(), device_types="cuda")
def embedding_backward(grad: torch.Tensor, tokens: torch.Tensor, vocabulary: int,
                       table_dtype: torch.dtype, position_dtype: torch.dtype, scale: float,
                       padding: int, need_table: bool, need_positions: bool
                       ) -> tuple[torch.Tensor, torch.Tensor]:
    """A gradient that is not needed comes back with 0 elements."""
    dtable, dpositions = _backward(grad, tokens, vocabulary, table_dtype, position_dtype, scale,
                                   padding, need_table, need_positions)
    return (grad.new_empty((0,), dtype=table_dtype) if dtable is None else dtable,
            grad.new_empty((0,), dtype=position_dtype) if dpositions is None else dpositions)


@embedding_backward.register_fake
def _(grad, tokens, vocabulary, table_dtype, position_dtype, scale, padding, need_table,
      need_positions):
    width = grad.shape[-1]
    period = tokens.shape[-1] if tokens.ndim else 1
    return (grad.new_empty((vocabulary, width) if need_table else (0,), dtype=table_dtype),
            grad.new_empty((period, width) if need_positions else (0,), dtype=position_dtype))


def _remember(ctx, tokens, table, positions, scale, padding) -> None:
    ctx.save_for_backward(tokens)
    ctx.set_materialize_grads(False)
    ctx.constants = (table.shape[0], table.dtype,
                     torch.float32 if positions is None else positions.dtype, scale, padding)


def _op_setup(ctx, inputs, output) -> None:
    tokens, table, positions, scale, padding, _dtype = inputs
    _remember(ctx, tokens, table, positions, scale, padding)


def _op_backward(ctx, grad):
    if grad is None:
        return (None,) * 6
    need = bool(ctx.needs_input_grad[1]), bool(ctx.needs_input_grad[2])
    grads = embedding_backward(grad, ctx.saved_tensors[0], *ctx.constants, *need)
    return (None, *(g if n else None for g, n in zip(grads, need)), None, None, None)


torch.library.register_autograd(embedding_forward, _op_backward, setup_context=_op_setup)


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, positions, scale, padding, dtype):
        _remember(ctx, tokens, table, positions, scale, padding)
        return _forward(tokens, table, positions, scale, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 6
        grads = _backward(grad, ctx.saved_tensors[0], *ctx.constants, *ctx.needs_input_grad[1:3])
        return (None, *grads, None, None, None)


def _check(tokens, table, positions, scale, padding_idx, dtype) -> None:
    _first_failure((
        (lambda: isinstance(tokens, torch.Tensor), TypeError, "tokens must be a tensor"),
        (lambda: isinstance(table, torch.Tensor), TypeError, "table must be a tensor"),
        (lambda: tokens.dtype in (torch.int64, torch.int32), TypeError,
         "tokens must be int64 or int32"),
        (lambda: table.dtype in _TYPES, TypeError, "table must be BF16, FP16 or FP32"),
        (lambda: dtype in _TYPES, TypeError, "dtype must be BF16, FP16 or FP32"),
        (lambda: tokens.device == table.device, TypeError, "tokens must be on the table's device"),
        (lambda: table.ndim == 2 and 1 <= table.shape[1] <= MAX_WIDTH, ValueError,
         f"expected table [V,D] with 1<=D<={MAX_WIDTH}"),
        (lambda: 1 <= table.shape[0] <= _calls.MAX_VOCABULARY, ValueError,
         f"supported vocabulary is 1<=V<={_calls.MAX_VOCABULARY}"),
        (lambda: tokens.numel() <= MAX_TOKENS, ValueError, "too many tokens"),
    ))
    if positions is not None:
        _first_failure((
            (lambda: isinstance(positions, torch.Tensor), TypeError, "positions must be a tensor"),
            (lambda: positions.dtype in _TYPES, TypeError, "positions must be BF16, FP16 or FP32"),
            (lambda: positions.device == table.device, TypeError,
             "positions must be on the table's device"),
            (lambda: positions.shape == (_period(tokens), table.shape[1]), ValueError,
             "positions must have shape [T,D], T the last axis of tokens"),
        ))
    check_scalar(scale, "scale")
    if padding_idx is not None:
        _first_failure((
            (lambda: isinstance(padding_idx, int) and not isinstance(padding_idx, bool), TypeError,
             "padding_idx must be an integer"),
            (lambda: -table.shape[0] <= padding_idx < table.shape[0], ValueError,
             "padding_idx must be an id of the table"),
        ))
    if not table.is_cuda:
        raise RuntimeError("embed requires CUDA tensors")


def embed(tokens: torch.Tensor, table: torch.Tensor, positions: torch.Tensor | None = None, *,
          scale: float = 1.0, padding_idx: int | None = None,
          dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * table[tokens] + positions``, summed in FP32 and rounded once to ``dtype``.

    ``tokens``: int64 or int32 ids ``[..., T]``; an id outside the table makes its row NaN (nothing
    is read out of range) and has no gradient.  ``table``: ``[V, D]``, ``positions``: ``[T, D]`` or
    None, each in BF16, FP16 or FP32; ``dtype`` defaults to the table's.  ``padding_idx`` names the
    id whose row gets no gradient (negative: from the end), as in ``F.embedding``.  The gradients of
    table (dense) and positions come back in their own types, summed in FP32 in the order of the
    tokens.  Differentiable once.
    """
    if dtype is None and isinstance(table, torch.Tensor):
        dtype = table.dtype
    _check(tokens, table, positions, scale, padding_idx, dtype)
    padding = -1 if padding_idx is None else padding_idx % table.shape[0]
    scale = float(scale)
    if not _calls.direct(tokens, table, positions):
        return embedding_forward(tokens, table, positions, scale, padding, dtype)
    if _calls.wants_grad(table, positions):
        return _Embed.apply(tokens, table, positions, scale, padding, dtype)
    return _forward(tokens, table, positions, scale, dtype)


__all__ = ["embed"]
