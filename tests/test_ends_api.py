"""Host-side contract of layer_norm, embed and linear_cross_entropy: what they refuse, in Python and
through the C ABI, found before any launch (no GPU needed)."""
import inspect

import pytest
import torch

from attnres import _native
from attnres.embedding import embed
from attnres.loss import linear_cross_entropy
from attnres.norm import layer_norm

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
X = torch.zeros(3, 16, dtype=BF16)
W = torch.ones(16)
IDS = torch.zeros(2, 3, dtype=torch.int64)
TABLE = torch.zeros(7, 16)
HEAD = torch.zeros(7, 16, dtype=BF16)
TARGETS = torch.zeros(3, dtype=torch.int64)


def test_signatures():
    assert list(inspect.signature(layer_norm).parameters) == ["x", "weight", "bias", "eps"]
    assert list(inspect.signature(embed).parameters) == [
        "tokens", "table", "positions", "scale", "padding_idx", "dtype"]
    assert list(inspect.signature(linear_cross_entropy).parameters) == [
        "hidden", "weight", "targets", "ignore_index", "reduction", "scale"]


@pytest.mark.parametrize("arguments,error,text", [
    ((X, W, W), RuntimeError, "CUDA"),
    ((X.double(),), TypeError, "BF16, FP16 or FP32"),
    (([1.0],), TypeError, "tensor"),
    ((torch.zeros((), dtype=BF16),), ValueError, "1<=D<=8192"),
    ((torch.zeros(2, 0),), ValueError, "1<=D<=8192"),
    ((torch.zeros(1, 8193),), ValueError, "1<=D<=8192"),
    ((X, W[:8]), ValueError, "weight must have shape"),
    ((X, W.double()), TypeError, "weight must be"),
    ((X, W, W[None]), ValueError, "bias must have shape"),
    ((X, 1.0), TypeError, "weight must be a tensor"),
    ((X, W, W, float("nan")), ValueError, "finite"),
    ((X, W, W, -1e-5), ValueError, "negative"),
    ((X, W, W, torch.tensor(1e-5)), TypeError, "real scalar"),
])
def test_layer_norm_refuses(arguments, error, text):
    with pytest.raises(error, match=text):
        layer_norm(*arguments)


@pytest.mark.parametrize("arguments,options,error,text", [
    ((IDS, TABLE), {}, RuntimeError, "CUDA"),
    ((IDS.float(), TABLE), {}, TypeError, "int64 or int32"),
    ((IDS.to(torch.int16), TABLE), {}, TypeError, "int64 or int32"),
    (([0], TABLE), {}, TypeError, "tokens must be a tensor"),
    ((IDS, [TABLE]), {}, TypeError, "table must be a tensor"),
    ((IDS, TABLE.double()), {}, TypeError, "table must be"),
    ((IDS, TABLE[0]), {}, ValueError, "expected table"),
    ((IDS, TABLE[:0]), {}, ValueError, "vocabulary"),
    ((IDS, torch.zeros(2, 8193)), {}, ValueError, "expected table"),
    ((IDS, TABLE), dict(dtype=torch.float64), TypeError, "dtype must be"),
    ((IDS, TABLE, TABLE[:2]), {}, ValueError, "positions must have shape"),
    ((IDS, TABLE, TABLE[:3].double()), {}, TypeError, "positions must be BF16"),
    ((IDS, TABLE), dict(scale=float("inf")), ValueError, "finite"),
    ((IDS, TABLE), dict(padding_idx=7), ValueError, "padding_idx"),
    ((IDS, TABLE), dict(padding_idx=-8), ValueError, "padding_idx"),
    ((IDS, TABLE), dict(padding_idx=1.0), TypeError, "padding_idx"),
])
def test_embed_refuses(arguments, options, error, text):
    with pytest.raises(error, match=text):
        embed(*arguments, **options)


@pytest.mark.parametrize("arguments,options,error,text", [
    ((X, HEAD, TARGETS), {}, RuntimeError, "CUDA"),
    ((X.float(), HEAD.float(), TARGETS), {}, TypeError, "BF16 or FP16"),
    ((X, HEAD.half(), TARGETS), {}, TypeError, "hidden's type"),
    ((X, HEAD, TARGETS.float()), {}, TypeError, "int64 or int32"),
    ((X, HEAD, 0), {}, TypeError, "must be tensors"),
    ((X, HEAD[:, :8], TARGETS), {}, ValueError, r"\[V,D\]"),
    ((X, HEAD[:0], TARGETS), {}, ValueError, "vocabulary"),
    ((X, HEAD, TARGETS[:2]), {}, ValueError, "leading axes"),
    ((X, HEAD, TARGETS), dict(reduction="batch"), ValueError, "reduction"),
    ((X, HEAD, TARGETS), dict(ignore_index=None), TypeError, "ignore_index"),
    ((X, HEAD, TARGETS), dict(scale=float("nan")), ValueError, "finite"),
    ((torch.zeros(3, 8200, dtype=BF16), HEAD, TARGETS), {}, ValueError, "8192"),
])
def test_linear_cross_entropy_refuses(arguments, options, error, text):
    with pytest.raises(error, match=text):
        linear_cross_entropy(*arguments, **options)


def test_norm_entry_points_check_their_arguments():
    lib = _native.load()

    def forward(x=0x1000, w=0x2000, b=0x3000, N=4, D=16, kind=0, param=2, eps=1e-5, y=0x4000):
        return lib.attnres_b200_norm_forward(x, D, w, b, N, D, kind, param, eps, y, None, None)

    assert forward(D=0) == 3 and forward(D=8193) == 3 and forward(N=0) == 5
    assert forward(kind=3) == 13 and forward(param=-1) == 13
    assert forward(eps=-1.0) == 6 and forward(eps=float("inf")) == 6
    assert forward(x=None) == 1 and forward(y=None) == 1
    assert forward(x=0x1001) == 7 and forward(w=0x2002) == 7 and forward(kind=2, y=0x4002) == 7

    def backward(g=0x1000, x=0x2000, stats=0x3000, dx=0x4000, partials=0x5000, dw=0x6000,
                 db=0x7000, N=4, D=16, kind=0):
        return lib.attnres_b200_norm_backward(g, D, x, D, stats, None, N, D, kind, 2, dx, partials,
                                              1 << 20, dw, db, None)

    assert backward(N=0) == 5 and backward(D=0) == 3 and backward(kind=9) == 13
    assert backward(g=None) == 1 and backward(stats=None) == 1 and backward(partials=None) == 1
    assert backward(dx=None, dw=None, db=None) == 11
    assert backward(dx=0x4001) == 7 and backward(dw=0x6002) == 7
    assert lib.attnres_b200_norm_workspace_rows(0, 16, 0) == -5
    assert lib.attnres_b200_norm_workspace_rows(4, 0, 0) == -3


def test_embedding_entry_points_check_their_arguments():
    lib = _native.load()

    def forward(tokens=0x1000, N=6, T=3, V=7, D=16, table=0x2000, kind=2, out=0x3000, out_kind=0,
                scale=1.0):
        return lib.attnres_b200_embedding_forward(tokens, 1, N, T, V, D, table, D, kind, None, 0, 2,
                                                  scale, out, out_kind, None)

    assert forward(N=0) == 5 and forward(T=4) == 5 and forward(N=1 << 31, T=1) == 5
    assert forward(V=0) == 14 and forward(V=(1 << 25) + 1) == 14
    assert forward(D=0) == 3 and forward(kind=7) == 13 and forward(scale=float("nan")) == 6
    assert forward(tokens=None) == 1 and forward(table=None) == 1 and forward(out=None) == 1
    assert forward(tokens=0x1004) == 7 and forward(table=0x2002) == 7 and forward(out=0x3001) == 7

    def backward(dtable=0x2000, dpos=0x3000, workspace=0x4000, size=1 << 40, N=6, T=3, grad=0x5000):
        return lib.attnres_b200_embedding_backward(0x1000, 1, N, T, 7, 16, -1, grad, 16, 0, 1.0,
                                                   dtable, 2, dpos, 2, workspace, size, None)

    assert backward(dtable=None, dpos=None) == 11
    assert backward(workspace=None) == 1 and backward(grad=None) == 1
    assert backward(workspace=0x4008) == 7 and backward(dtable=0x2001) == 7
    assert backward(size=64) == 8 and backward(N=7) == 5
    assert lib.attnres_b200_embedding_workspace_bytes(0, 16) == -5
    assert lib.attnres_b200_embedding_workspace_bytes(6, 0) == -3
    assert lib.attnres_b200_embedding_workspace_bytes(6, 16) >= 6 * 16


def test_loss_entry_points_check_their_arguments():
    lib = _native.load()

    def forward(N=3, V=7, D=16, kind=0, scale=1.0, reduction=2, hidden=0x1000, weight=0x2000,
                targets=0x3000, kept=0x4000, loss=0x5000, workspace=0x6000, size=1 << 40, sums=0x7300,
                dh=None, dw=None):
        return lib.attnres_b200_loss_forward(hidden, D, weight, D, targets, 1, N, V, D, kind, -100,
                                             scale, reduction, kept, 0x7000, 0x7100, 0x7200, sums,
                                             0x7400, loss, dh, dw, workspace, size, None)

    assert forward(N=0) == 5 and forward(D=8193) == 3 and forward(V=0) == 14
    assert forward(kind=2) == 13 and forward(scale=float("inf")) == 6 and forward(reduction=3) == 10
    assert forward(hidden=None) == 1 and forward(kept=None) == 1 and forward(loss=None) == 1
    assert forward(hidden=0x1001) == 7 and forward(kept=0x4008) == 7 and forward(targets=0x3004) == 7
    assert forward(size=16) == 8 and forward(sums=None) == 1
    # gradients in the forward: BF16 and one loss
    assert forward(dh=0x8000, kind=1) == 13 and forward(dw=0x8000, reduction=0) == 10
    assert forward(dh=0x8001) == 7 and forward(dh=0x8000, sums=None, size=16) == 8

    def backward(dh=0x1000, dw=0x2000, upstream=0x3000, workspace=0x6000, size=1 << 40, kind=0):
        return lib.attnres_b200_loss_backward(upstream, 1, 0x2000, 16, 0x3000, 1, 3, 7, 16, kind,
                                              -100, 1.0, 2, 0x4000, 0x7000, 0x7100, 0x7200, 0x7300,
                                              dh, dw, workspace, size, None)

    assert backward(dh=None, dw=None) == 11 and backward(upstream=None) == 1
    assert backward(dh=0x1001) == 7 and backward(workspace=0x6008) == 7
    assert backward(size=16) == 8 and backward(kind=2) == 13
    assert lib.attnres_b200_loss_workspace_bytes(0, 7, 16, 0) == -5
    assert lib.attnres_b200_loss_workspace_bytes(3, 0, 16, 1) == -14
    # a piece of the vocabulary, not the vocabulary: 16 384 x 128 000 logits would be 4 GB
    assert lib.attnres_b200_loss_workspace_bytes(16384, 128000, 64, 1) < 1200 << 20
    assert lib.attnres_b200_loss_workspace_bytes(16384, 128000, 64, 2) < 1300 << 20
    assert lib.attnres_b200_loss_workspace_bytes(3, 7, 16, 3) == -10
    policy = lib.attnres_b200_loss_gradients_in_forward
    assert policy(512, 0, 2) and policy(1024, 0, 1)
    assert not policy(511, 0, 2) and not policy(1024, 1, 2) and not policy(1024, 0, 0)

    def scaled(gradient=0x1000, upstream=0x2000, count=8, out=0x3000):
        return lib.attnres_b200_loss_scale_gradient(gradient, upstream, count, out, None)

    assert scaled(count=0) == 5 and scaled(gradient=None) == 1 and scaled(upstream=None) == 1
    assert scaled(gradient=0x1008) == 7 and scaled(out=0x3002) == 7
