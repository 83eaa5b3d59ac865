"""What the compiled operators (norm, embedding, loss) share on the Python side."""
from __future__ import annotations

import torch

FLOATS = frozenset((torch.bfloat16, torch.float16, torch.float32))
HALVES = frozenset((torch.bfloat16, torch.float16))
INTEGERS = frozenset((torch.int64, torch.int32))
MAX_VOCABULARY = 1 << 25


def plain_number(value) -> bool:
    """An int or float: the common case of ``check_scalar``, which judges everything else."""
    return type(value) is float or type(value) is int
