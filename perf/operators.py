"""Cases, plain forms and 64-bit values of the operators at the two ends of an AttnRes network.

Between its token ids and its loss a network of AttnRes reads runs three operators that are not
reads: the embedding that makes the first source, the LayerNorm in front of the first sublayer
(every later sublayer has its norm in the read's epilogue) and the loss over the vocabulary that
consumes the last read.  This file says at which sizes they are measured and what they compute:

* ``norm``   y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, and its gradients;
* ``embed``  out[b, t] = scale * table[token[b, t]] + positions[t], and its gradients;
* ``loss``   softmax cross entropy of ``scale * hidden @ weight.T`` against target ids, rows with
  the ignored id left out, and the gradients of hidden and weight.

``run`` computes them from elementary torch operations in 32 bits (``own = False``) or through the
library's entry points (``own = True``); ``exact`` from their definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORED = -100


def listed():
    return [
        # The norm of a few rows: one decoding step of eight sequences at the wide model's width.
        dict(name="norm_step_8x4096", op="norm", rows=8, width=4096, type="bf16", weights="bf16",
             affine="both", pad=0, train=False),
        # The first sublayer's norm in a training step of the 24-layer, 1024-wide model: 8 x 2048
        # positions, FP32 parameters under BF16 autocast.
        dict(name="norm_train_16384x1024", op="norm", rows=16384, width=1024, type="bf16",
             weights="fp32", affine="both", pad=0, train=True),
        # Odd sizes: an FP32 stream with rows that are slices of a wider buffer, no bias.
        dict(name="norm_train_fp32_4099x1537", op="norm", rows=4099, width=1537, type="fp32",
             weights="fp32", affine="weight", pad=3, train=True),
        # The same norm in the 4096-wide model, BF16 parameters, a microbatch of 4 x 4096.
        dict(name="norm_train_16384x4096", op="norm", rows=16384, width=4096, type="bf16",
             weights="bf16", affine="both", pad=0, train=True),
        # The embedding of one decoding step.
        dict(name="embed_step_16x4096", op="embed", batch=1, length=16, vocab=32000, width=4096,
             type="bf16", out="bf16", scale=1.0, positions=False, padding=False, skew=0.0,
             train=False),
        # The 1024-wide model's first source: FP32 table and positions, BF16 result, uniform ids.
        dict(name="embed_train_8x2048x1024", op="embed", batch=8, length=2048, vocab=32000,
             width=1024, type="fp32", out="bf16", scale=1.0, positions=True, padding=False,
             skew=0.0, train=True),
        # Odd sizes: padded sequences of text-like ids (a few are most of them), scaled by sqrt(D).
        dict(name="embed_train_5x1237x1001", op="embed", batch=5, length=1237, vocab=50021,
             width=1001, type="fp16", out="fp16", scale=31.64, positions=False, padding=True,
             skew=1.0, train=True),
        # The 4096-wide model's first source on text-like ids, BF16 parameters.
        dict(name="embed_train_4x4096x4096", op="embed", batch=4, length=4096, vocab=32000,
             width=4096, type="bf16", out="bf16", scale=1.0, positions=True, padding=False,
             skew=1.0, train=True),
        # Scoring a short continuation: the loss of each of 64 positions, no gradients.
        dict(name="loss_score_64x32000x1024", op="loss", rows=64, vocab=32000, width=1024,
             type="bf16", scale=1.0, ignored=0.0, reduction="none", train=False),
        # Odd sizes: fine-tuning on answers only (prompt positions ignored), FP16, odd vocabulary.
        dict(name="loss_train_1531x10007x523", op="loss", rows=1531, vocab=10007, width=523,
             type="fp16", scale=1.0, ignored=0.4, reduction="sum", train=True),
        # The 1024-wide model's head and loss over a whole step.
        dict(name="loss_train_16384x32000x1024", op="loss", rows=16384, vocab=32000, width=1024,
             type="bf16", scale=1.0, ignored=0.0, reduction="mean", train=True),
        # The 4096-wide model's head and loss over one microbatch, some positions padded.
        dict(name="loss_train_16384x32000x4096", op="loss", rows=16384, vocab=32000, width=4096,
             type="bf16", scale=1.0, ignored=0.1, reduction="mean", train=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "embed", "loss"])
    train = rng.random() < 0.7
    if op == "norm":
        width = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(65536, 16384 * 4096 // width))
        return dict(op=op, rows=rows, width=width, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    weights=rng.choice(["fp32", "bf16"]),
                    affine=rng.choice(["both", "both", "weight", "none"]),
                    pad=rng.choice([0, 0, 8, 3]), train=train)
    if op == "embed":
        width = _log_int(rng, 16, 8192)
        vocab = _log_int(rng, 2, min(131072, 32000 * 4096 // width))
        count = _log_int(rng, 1, min(65536, 16384 * 4096 // width))
        batch = rng.choice([b for b in (1, 2, 3, 5, 8) if b <= count])
        kind = rng.choice(["bf16", "fp16", "fp32"])
        return dict(op=op, batch=batch, length=count // batch, vocab=vocab, width=width, type=kind,
                    out=rng.choice(["bf16", kind]), scale=rng.choice([1.0, math.sqrt(width)]),
                    positions=rng.random() < 0.5, padding=rng.random() < 0.3,
                    skew=rng.choice([0.0, 1.0]), train=train)
    width = _log_int(rng, 16, 4096)
    vocab = _log_int(rng, 2, 131072)
    rows = _log_int(rng, 1, max(1, min(32768, 16384 * 32000 // vocab)))
    return dict(op=op, rows=rows, vocab=vocab, width=width, type=rng.choice(["bf16", "bf16", "fp16"]),
                scale=rng.choice([1.0, 1.0, 0.5]), ignored=rng.choice([0.0, 0.1, 0.4]),
                reduction=rng.choice(["mean", "sum", "none"]), train=train)


# ------------------------------------------------------------------------------------- inputs

def _normal(generator, shape, kind, spread=1.0, centre=0.0):
    x = torch.empty(shape, device="cuda", dtype=torch.float32)
    x.normal_(centre, spread, generator=generator)
    return x.to(_TYPES[kind])


def _ids(generator, count, vocab, skew):
    """Uniform ids, or ids whose frequency falls as 1 / rank with the ranks shuffled."""
    if not skew:
        return torch.randint(vocab, (count,), device="cuda", generator=generator)
    u = torch.rand(count, device="cuda", generator=generator, dtype=torch.float64)
    ranks = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return torch.randperm(vocab, device="cuda", generator=generator)[ranks]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 40))
    state = dict(case)
    if case["op"] == "norm":
        rows, width, kind = case["rows"], case["width"], case["type"]
        x = _normal(generator, (rows, width + case["pad"]), kind, 1.5, 0.3)[:, :width]
        weight = _normal(generator, (width,), case["weights"], 0.1, 1.0)
        bias = _normal(generator, (width,), case["weights"], 0.1)
        state.update(x=x, weight=weight if case["affine"] != "none" else None,
                     bias=bias if case["affine"] == "both" else None)
        state["upstream"] = _normal(generator, (rows, width), kind)
        leaves = [x, state["weight"], state["bias"]]
    elif case["op"] == "embed":
        count = case["batch"] * case["length"]
        tokens = _ids(generator, count, case["vocab"], case["skew"])
        state["padding_idx"] = None
        if case["padding"]:   # the last quarter of every sequence
            state["padding_idx"] = 0
            tokens.view(case["batch"], case["length"])[:, case["length"] * 3 // 4:] = 0
        state["tokens"] = tokens.view(case["batch"], case["length"])
        table = _normal(generator, (case["vocab"], case["width"]), case["type"], 0.02)
        positions = _normal(generator, (case["length"], case["width"]), case["type"], 0.02)
        state.update(table=table, position_rows=positions if case["positions"] else None)
        state["upstream"] = _normal(generator, (case["batch"], case["length"], case["width"]),
                                    case["out"])
        leaves = [table, state["position_rows"]]
    else:
        rows, vocab, width = case["rows"], case["vocab"], case["width"]
        weight = _normal(generator, (vocab, width), case["type"], 1.0 / math.sqrt(width))
        targets = torch.randint(vocab, (rows,), device="cuda", generator=generator)
        # Half learned: the target's logit stands out by a few units, more in some rows.
        lift = torch.rand(rows, 1, device="cuda", generator=generator) * 8.0
        hidden = _normal(generator, (rows, width), "fp32") + lift * weight[targets].float()
        if case["ignored"]:
            drop = torch.rand(rows, device="cuda", generator=generator) < case["ignored"]
            drop[0] = False
            targets = torch.where(drop, torch.full_like(targets, IGNORED), targets)
        hidden = hidden.to(_TYPES[case["type"]])
        state.update(hidden=hidden, weight=weight, targets=targets, upstream=None)
        if case["reduction"] == "none":
            state["upstream"] = torch.rand(rows, device="cuda", generator=generator) + 0.5
        leaves = [hidden, weight]
    state["leaves"] = [leaf.requires_grad_(case["train"]) for leaf in leaves if leaf is not None]
    return state


# ------------------------------------------------------------------------------------- one pass

_calls = {}


def _library():
    if not _calls:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                               "fast-attnres_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from attnres.embedding import embed
        from attnres.loss import linear_cross_entropy
        from attnres.norm import layer_norm
        _calls.update(norm=layer_norm, embed=embed, loss=linear_cross_entropy)
    return _calls


def run(state):
    if own:
        return _run_library(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "embed": _plain_embed, "loss": _plain_loss}[state["op"]](state)


def _run_library(state):
    op = state["op"]
    call = _library()[op]
    if op == "norm":
        result = call(state["x"], state["weight"], state["bias"], 1e-5)
    elif op == "embed":
        result = call(state["tokens"], state["table"], state["position_rows"], scale=state["scale"],
                      padding_idx=state["padding_idx"], dtype=_TYPES[state["out"]])
    else:
        result = call(state["hidden"], state["weight"], state["targets"], ignore_index=IGNORED,
                      reduction=state["reduction"], scale=state["scale"])
    if not state["train"]:
        return [result]
    return [result.detach(), *torch.autograd.grad(result, state["leaves"], state["upstream"])]


def _plain_norm(state):
    x = state["x"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    unit = centred * rstd
    weight, bias = state["weight"], state["bias"]
    y = unit
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    outputs = [y.to(state["x"].dtype)]
    if state["train"]:
        upstream = state["upstream"].float()
        g = upstream if weight is None else upstream * weight.float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
        outputs.append(dx.to(state["x"].dtype))
        if weight is not None:
            outputs.append((upstream * unit).sum(0).to(weight.dtype))
        if bias is not None:
            outputs.append(upstream.sum(0).to(bias.dtype))
    return outputs


def _plain_embed(state):
    tokens, table, positions = state["tokens"], state["table"], state["position_rows"]
    out = table[tokens].float() * state["scale"]
    if positions is not None:
        out = out + positions.float()
    outputs = [out.to(_TYPES[state["out"]])]
    if state["train"]:
        upstream = state["upstream"].float()
        rows = upstream * state["scale"]
        if state["padding_idx"] is not None:
            rows = torch.where((tokens != state["padding_idx"])[..., None], rows, 0.0)
        grad = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
        grad.index_add_(0, tokens.reshape(-1), rows.reshape(-1, rows.shape[-1]))
        outputs.append(grad.to(table.dtype))
        if positions is not None:
            outputs.append(upstream.sum(0).to(positions.dtype))
    return outputs


def _plain_loss(state):
    hidden, weight, targets = state["hidden"].float(), state["weight"].float(), state["targets"]
    kept = targets != IGNORED
    ids = torch.where(kept, targets, 0)[:, None]
    z = hidden @ weight.t() * state["scale"]
    e = z - z.amax(-1, keepdim=True)
    at_target = e.gather(1, ids)[:, 0]
    e = e.exp()
    total = e.sum(-1, keepdim=True)
    losses = torch.where(kept, total[:, 0].log() - at_target, 0.0)
    count = kept.sum()
    if state["reduction"] == "none":
        loss, coefficient = losses, state["upstream"]
    elif state["reduction"] == "sum":
        loss, coefficient = losses.sum(), 1.0
    else:
        loss, coefficient = losses.sum() / count, 1.0 / count
    if not state["train"]:
        return [loss]
    p = e / total
    p.scatter_add_(1, ids, torch.full_like(ids, -1, dtype=p.dtype))
    p = p * torch.where(kept, coefficient * state["scale"], 0.0)[:, None]
    return [loss, (p @ weight).to(state["hidden"].dtype), (p.t() @ hidden).to(state["weight"].dtype)]


# ------------------------------------------------------------------------------------- accounts

def work(case):
    """Each input once, each output once; products of the definition, the logits formed once."""
    if case["op"] == "norm":
        cells, size = case["rows"] * case["width"], _BYTES[case["type"]]
        parameters = {"both": 2, "weight": 1, "none": 0}[case["affine"]] * case["width"]
        parameters *= _BYTES[case["weights"]]
        if not case["train"]:
            return {"bytes": 2 * cells * size + parameters, "flops": 8 * cells}
        return {"bytes": 4 * cells * size + 2 * parameters, "flops": 24 * cells}
    if case["op"] == "embed":
        count, width = case["batch"] * case["length"], case["width"]
        size, out = _BYTES[case["type"]], _BYTES[case["out"]]
        touched = case["vocab"] * -math.expm1(-count / case["vocab"])   # distinct ids, if uniform
        if case["skew"]:   # sum over ranks of 1 - exp(-expected uses)
            ranks = torch.arange(case["vocab"], dtype=torch.float64)
            share = torch.log1p(1.0 / (ranks + 1.0)) / math.log(case["vocab"] + 1.0)
            touched = float(-torch.expm1(-count * share).sum())
        held = case["length"] * width * size if case["positions"] else 0
        moved = count * 8 + touched * width * size + held + count * width * out
        if case["train"]:
            moved += count * width * out + case["vocab"] * width * size + held
        return {"bytes": moved, "flops": (4 if case["train"] else 2) * count * width}
    rows = case["rows"] * (1.0 - case["ignored"])
    size, product = _BYTES[case["type"]], 2.0 * rows * case["vocab"] * case["width"]
    held = (rows + case["vocab"]) * case["width"] * size + case["rows"] * 8
    if not case["train"]:
        return {"bytes": held + 4 * case["rows"], "flops": product + 4 * rows * case["vocab"]}
    wide = (case["rows"] + case["vocab"]) * case["width"] * size
    return {"bytes": held + wide + 4, "flops": 3 * product + 8 * rows * case["vocab"]}


# ------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: (v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v)
            for k, v in state.items()}
    return {"norm": _exact_norm, "embed": _exact_embed, "loss": _exact_loss}[case["op"]](wide)


def _exact_norm(state):
    """Row by row through autograd: the definition with the population variance."""
    leaves = [t.requires_grad_() for t in (state["x"], state["weight"], state["bias"])
              if t is not None]
    with torch.enable_grad():
        variance, mean = torch.var_mean(state["x"], -1, correction=0, keepdim=True)
        y = (state["x"] - mean) / (variance + 1e-5).sqrt()
        if state["weight"] is not None:
            y = y * state["weight"]
        if state["bias"] is not None:
            y = y + state["bias"]
    if not state["train"]:
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["upstream"])]


def _exact_embed(state):
    """The table's gradient as sums over runs of equal ids, by differences of prefix counts."""
    tokens, table = state["tokens"], state["table"]
    out = torch.mul(torch.index_select(table, 0, tokens.flatten()), state["scale"])
    out = out.view(*tokens.shape, -1)
    if state["position_rows"] is not None:
        out = out + state["position_rows"][None]
    if not state["train"]:
        return [out]
    flat, upstream = tokens.flatten(), state["upstream"].flatten(0, 1) * state["scale"]
    used = torch.ones_like(flat, dtype=torch.bool)
    if state["padding_idx"] is not None:
        used = flat != state["padding_idx"]
    one_hot = torch.sparse_coo_tensor(
        torch.stack((flat[used], torch.arange(flat.numel(), device=flat.device)[used])),
        torch.ones(int(used.sum()), device=flat.device, dtype=torch.float64),
        (table.shape[0], flat.numel()))
    outputs = [out, torch.sparse.mm(one_hot, upstream)]
    if state["position_rows"] is not None:
        outputs.append(state["upstream"].sum(0))
    return outputs


def _exact_loss(state):
    """A slice of the rows at a time: log-sum-exp, then (softmax - one-hot) against both factors."""
    hidden, weight, targets = state["hidden"], state["weight"], state["targets"]
    rows, scale = hidden.shape[0], state["scale"]
    valid = targets.ge(0)
    coefficient = torch.ones(rows, device=hidden.device, dtype=torch.float64)
    if state["reduction"] == "mean":
        coefficient /= valid.sum()
    elif state["reduction"] == "none" and state["upstream"] is not None:
        coefficient = state["upstream"].clone()
    coefficient[~valid] = 0.0
    losses = torch.zeros(rows, device=hidden.device, dtype=torch.float64)
    dhidden, dweight = torch.zeros_like(hidden), torch.zeros_like(weight)
    for first in range(0, rows, 4096):
        part = slice(first, min(rows, first + 4096))
        logits = scale * torch.einsum("nd,vd->nv", hidden[part], weight)
        normaliser = torch.logsumexp(logits, 1)
        one_hot = torch.arange(weight.shape[0], device=targets.device) == targets[part, None]
        losses[part] = normaliser - torch.where(one_hot, logits, 0.0).sum(1)
        if state["train"]:
            residue = torch.softmax(logits, 1).sub_(one_hot.double())
            residue *= scale * coefficient[part, None]
            dhidden[part] = residue @ weight
            dweight += residue.t() @ hidden[part]
    losses = torch.where(valid, losses, 0.0)
    loss = losses
    if state["reduction"] != "none":
        loss = losses.sum() / (valid.sum() if state["reduction"] == "mean" else 1)
    return [loss, dhidden, dweight] if state["train"] else [loss]
