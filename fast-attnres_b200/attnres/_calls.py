"""Shared plumbing of the operators at the ends of the network (norm, embedding, loss).

These operators also run on a handful of rows, where the host's share of a call is most of its
time, so each has two ways to the same C-ABI call: under ``torch.compile`` (and any tensor subclass
or dispatch mode) it is a ``torch.library`` operator with a fake kernel and registered autograd;
an eager call on plain tensors goes through an ``autograd.Function``, or straight to the launch
when no gradient is wanted, which costs a third of the operator's dispatch.
"""
from __future__ import annotations

import contextlib

import torch
from torch.utils._python_dispatch import _get_current_dispatch_mode

TYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_HERE = contextlib.nullcontext()
MAX_VOCABULARY = 1 << 25


def direct(*tensors) -> bool:
    """Whether a call may skip the operator dispatcher: eager, plain tensors, no dispatch mode."""
    if torch.compiler.is_compiling() or _get_current_dispatch_mode() is not None:
        return False
    return all(t is None or type(t) in _PLAIN for t in tensors)


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def on_device(device: torch.device):
    """A context in which `device` is current; free when it already is."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def pointer(tensor):
    return None if tensor is None else tensor.data_ptr()


def rows_of(tensor: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(tensor, row stride) with feature stride 1: `tensor` itself where its leading axes can be
    walked with one stride, a contiguous copy otherwise."""
    if tensor.is_contiguous():
        return tensor, tensor.shape[-1]
    from ._sources import row_layout
    kept, row_stride, feature_stride = row_layout(tensor)
    if feature_stride != 1 and kept.shape[-1] > 1:
        kept = kept.contiguous()
        row_stride = kept.shape[-1]
    return kept, row_stride
