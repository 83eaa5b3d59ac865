"""The operators at the two ends of a network of reads: the embedding that makes the first source,
the LayerNorm of a sublayer that no read precedes, and the head with its loss, whose logits never
exist.  Needs a CUDA device.

    python fast-attnres_b200/examples/network_ends.py
"""
from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402
import torch.nn.functional as F  # noqa: E402

from attnres import attnres  # noqa: E402
from attnres.embedding import embed  # noqa: E402
from attnres.loss import linear_cross_entropy  # noqa: E402
from attnres.norm import layer_norm  # noqa: E402


def run(device: str = "cuda") -> dict:
    torch.manual_seed(4)
    batch, length, vocabulary, width = 4, 96, 5000, 512
    table = (0.5 * torch.randn(vocabulary, width, device=device)).requires_grad_()
    positions = (0.1 * torch.randn(length, width, device=device)).requires_grad_()
    norm = torch.nn.LayerNorm(width).to(device)
    mix = torch.nn.Linear(width, width, bias=False, device=device, dtype=torch.bfloat16)
    query = (0.1 * torch.randn(width, device=device)).to(torch.bfloat16).requires_grad_()
    head = (torch.randn(vocabulary, width, device=device) / width**0.5).to(torch.bfloat16).requires_grad_()
    tokens = torch.randint(vocabulary, (batch, length), device=device)
    targets = torch.roll(tokens, -1, dims=1)
    targets[:, -1] = -100                     # nothing follows the last token
    leaves = (table, positions, norm.weight, norm.bias, mix.weight, query, head)

    # the whole network on this library: ids -> first source -> sublayer -> read -> loss
    first = embed(tokens, table, positions, dtype=torch.bfloat16)
    second = mix(layer_norm(first, norm.weight, norm.bias, norm.eps))
    loss = linear_cross_entropy(attnres((first, second), query), head, targets)
    grads = torch.autograd.grad(loss, leaves)

    # the same from the framework's own pieces, logits and all
    first = (F.embedding(tokens, table) + positions).to(torch.bfloat16)
    second = mix(F.layer_norm(first.float(), (width,), norm.weight, norm.bias, norm.eps).to(torch.bfloat16))
    logits = (attnres((first, second), query) @ head.t()).float()
    expected = F.cross_entropy(logits.reshape(-1, vocabulary), targets.reshape(-1))
    wanted = torch.autograd.grad(expected, leaves)

    torch.testing.assert_close(loss, expected, rtol=2**-8, atol=0)
    for got, want in zip(grads, wanted):
        error = (got.float() - want.float()).norm() / want.float().norm()
        assert error < 2**-5, error
    return {"loss": float(loss), "gradients": len(grads)}


if __name__ == "__main__":
    print(run())
