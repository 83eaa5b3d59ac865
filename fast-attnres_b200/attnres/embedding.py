"""Embedding lookup with scaling and learned positions: the first source of a network of reads.

The reference's model adds a token row and a position row and casts the sum to the working type of
the stream (benchmarks/model.py:239-245 of the reference): three passes over ``[N, D]``, and a
table gradient that is scattered with atomics.  Here the lookup, the scale, the positions and the
cast are one pass, and the gradient of the table is a sum over the tokens sorted by id, in a fixed
order, so it is the same bits every time.

    first = embed(tokens, table, positions[:tokens.shape[-1]], dtype=torch.bfloat16)
"""
from __future__ import annotations

import math

import torch

from . import _calls, _native
from ._sources import MAX_WIDTH, _first_failure, check_scalar

# Compiled operators (csrc/torch_ops.cpp): `embedding_forward` and `embedding_backward` launch the
# kernels, `embed` is the differentiable call over the two.
_ops = _native.load_operators()
_embed = _ops.embed.default
_TYPES = _calls.FLOATS
MAX_TOKENS = 2**31 - 1


def _period(tokens) -> int:
    return tokens.shape[-1] if tokens.ndim else 1


@torch.library.register_fake("attnres_b200::embedding_forward")
def _(tokens, table, positions, scale, type):
    return table.new_empty((*tokens.shape, table.shape[1]), dtype=type)


@torch.library.register_fake("attnres_b200::embedding_backward")
def _(grad, tokens, vocabulary, table_type, position_type, scale, padding, need_table,
      need_positions):
    width = grad.shape[-1]
    return (grad.new_empty((vocabulary, width) if need_table else (0,), dtype=table_type),
            grad.new_empty((_period(tokens), width) if need_positions else (0,),
                           dtype=position_type))


@torch.library.register_fake("attnres_b200::embed")
def _(tokens, table, positions, scale, padding, type):
    return table.new_empty((*tokens.shape, table.shape[1]), dtype=type)


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


def _acceptable(tokens, table, dtype) -> bool:
    """The conditions of `_check` at the cost of a call on a few tokens; `_check` names the one
    that does not hold."""
    return (isinstance(tokens, torch.Tensor) and isinstance(table, torch.Tensor) and table.is_cuda
            and tokens.dtype in _calls.INTEGERS and table.dtype in _TYPES and dtype in _TYPES
            and tokens.device == table.device and table.ndim == 2
            and 1 <= table.shape[1] <= MAX_WIDTH and 1 <= table.shape[0] <= _calls.MAX_VOCABULARY
            and tokens.numel() <= MAX_TOKENS)


def _positions_ok(positions, tokens, table) -> bool:
    return (isinstance(positions, torch.Tensor) and positions.dtype in _TYPES
            and positions.device == table.device and positions.ndim == 2
            and positions.shape[0] == _period(tokens) and positions.shape[1] == table.shape[1])


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
    if not (_acceptable(tokens, table, dtype)
            and (positions is None or _positions_ok(positions, tokens, table))
            and _calls.plain_number(scale) and math.isfinite(scale)
            and (padding_idx is None or (type(padding_idx) is int
                                         and -table.shape[0] <= padding_idx < table.shape[0]))):
        _check(tokens, table, positions, scale, padding_idx, dtype)
    padding = -1 if padding_idx is None else padding_idx % table.shape[0]
    return _embed(tokens, table, positions, scale, padding, dtype)


__all__ = ["embed"]
