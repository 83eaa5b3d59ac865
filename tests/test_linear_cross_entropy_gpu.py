"""linear_cross_entropy against its definition in 64 bits, forward and backward.

Tolerances, with e = 2^-23 (a step of FP32) and h half a step of the inputs' type:
  a logit, D products added in FP32 on the tensor cores (16 at a time, each addition off by at most
  two steps of the running sum): cz = (D/8 + 16) e max_v sum_d |h w|, times |scale|;
  a loss is off by 2 cz and, from the exponentials and logarithms, 8 e (1 + |lse| + |z|);
  a probability by a factor 1 + cp, cp = 2 cz + 8 e (1 + |lse|); the residue P = c (p - onehot) is
  rounded once to the inputs' type, so |dP| <= h |P| + cp c p;
  a gradient is a sum of V (or N) products: (V/8 + 16) e sum |P||W| on top, and rounded once.
FP16 keeps P as 2^15 P / max c: half of its smallest subnormal is 2^-40 max c in P.
BF16 keeps P / max c, and the exponential of a logit that lies more than 126 powers of two below the
row's sum is zero (FP32 has no normal number for it): 2^-126 max c in P, whatever P's own size.
Where the forward forms the gradients (BF16, a sum or mean, 512 features and more) a logit passes
through a code in steps of 2^-11 powers of two below its half tile's maximum, 65535 of them at most:
a probability is off by a factor 2^(+-2^-12), less than 2^-12, or is 2^-32 of that maximum instead of
something smaller; and the gradient is rounded once more when the upstream gradient multiplies it.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0**-23


def _case(rows, vocabulary, width, dtype, *, ignored=0.0, seed=0, lift=4.0):
    generator = torch.Generator(device="cuda").manual_seed(seed + 7919 * rows + vocabulary)
    weight = torch.randn(vocabulary, width, device="cuda", generator=generator) / math.sqrt(width)
    weight = weight.to(dtype)
    targets = torch.randint(vocabulary, (rows,), device="cuda", generator=generator)
    hidden = torch.randn(rows, width, device="cuda", generator=generator)
    hidden = hidden + lift * torch.rand(rows, 1, device="cuda", generator=generator) * weight[targets].float()
    if ignored:
        targets[torch.rand(rows, device="cuda", generator=generator) < ignored] = -100
    return hidden.to(dtype), weight, targets


def _reference(hidden, weight, targets, reduction, scale, upstream, ignore_index):
    h, w = hidden.detach().double(), weight.detach().double()
    rows, width = h.shape
    vocabulary = w.shape[0]
    half = torch.finfo(hidden.dtype).eps / 2
    kept = targets != ignore_index
    ids = torch.where(kept, targets, 0).long()
    h = torch.where(kept[:, None], h, 0.0)
    z = scale * h @ w.t()
    cz = (width / 8 + 16) * E * abs(scale) * (h.abs() @ w.abs().t()).amax(1)
    lse = z.logsumexp(1)
    at = z.gather(1, ids[:, None])[:, 0]
    losses = torch.where(kept, lse - at, 0.0)
    loss_slack = torch.where(kept, 2 * cz + 8 * E * (1 + lse.abs() + at.abs()), 0.0)
    count = kept.sum()
    if reduction == "none":
        loss, slack, c = losses, loss_slack, upstream.double()
    elif reduction == "sum":
        loss, slack, c = losses.sum(), loss_slack.sum(), upstream.double().expand(rows)
    else:
        loss, slack, c = losses.sum() / count, loss_slack.sum() / count, (upstream.double() / count).expand(rows)
    c = torch.where(kept, c, 0.0)[:, None] * scale
    p = (z - lse[:, None]).exp()
    cp = (2 * cz + 8 * E * (1 + lse.abs()))[:, None]
    spread = c.abs() * p * cp
    early = hidden.dtype == BF16 and reduction != "none" and width >= 512
    if early:
        spread += c.abs() * (2.0**-12 * p + 2.0**-32)
    p.scatter_add_(1, ids[:, None], torch.full_like(p[:, :1], -1.0))
    p *= c
    spread += half * p.abs()
    spread += (2.0**-40 if hidden.dtype == FP16 else 2.0**-126) * c.abs().max() * kept[:, None]
    size = p.abs() + spread
    dhidden, dweight = p @ w, p.t() @ h
    again = half if early else 0.0
    return dict(
        loss=(loss, slack),
        dhidden=(dhidden, again * dhidden.abs() + (1 + again) * (
            spread @ w.abs() + (vocabulary / 8 + 24) * E * (size @ w.abs()))),
        dweight=(dweight, again * dweight.abs() + (1 + again) * (
            spread.t() @ h.abs() + (rows / 8 + 24) * E * (size.t() @ h.abs()))))


def _inside(got, want, slack, what):
    info = torch.finfo(got.dtype)
    assert got.shape == want.shape, what
    assert got.isfinite().all(), what
    off = (got.double() - want).abs()
    limit = info.eps / 2 * (want.abs() + slack) + slack + info.smallest_normal * info.eps / 2
    assert not (off > limit).any().item(), (what, off.max().item(), (off / limit).max().item())


def _check(hidden, weight, targets, *, reduction="mean", scale=1.0, upstream=None, ignore_index=-100):
    from attnres.loss import linear_cross_entropy
    call = lambda: linear_cross_entropy(hidden, weight, targets, reduction=reduction,  # noqa: E731
                                        scale=scale, ignore_index=ignore_index)
    width = hidden.shape[-1]
    if upstream is None:
        upstream = torch.ones(targets.shape if reduction == "none" else (), device="cuda")
    want = _reference(hidden.reshape(-1, width), weight, targets.reshape(-1), reduction, scale,
                      upstream.reshape(-1) if reduction == "none" else upstream, ignore_index)
    with torch.no_grad():
        alone = call()
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    loss = call()
    assert loss.dtype == FP32 and torch.equal(loss, alone)
    assert loss.shape == (targets.shape if reduction == "none" else ())
    grads = torch.autograd.grad(loss, leaves, upstream)
    _inside(loss.detach().reshape(want["loss"][0].shape), *want["loss"], "loss")
    _inside(grads[0].reshape(-1, width), *want["dhidden"], "dhidden")
    _inside(grads[1], *want["dweight"], "dweight")
    assert grads[0].dtype == hidden.dtype and grads[1].dtype == weight.dtype
    return loss.detach(), *grads


# one row, one word, sizes around the tile (128 rows, 256 words, 64 columns), odd widths
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,vocabulary,width", [
    (1, 1, 8), (1, 2, 1), (2, 31, 16), (7, 300, 64), (128, 256, 64), (127, 255, 63), (129, 257, 65),
    (200, 1000, 128), (333, 777, 523), (256, 512, 1024), (65, 5003, 200), (1000, 130, 72),
    (40, 128, 4096), (3, 9, 8192), (5, 40000, 24)])
def test_linear_cross_entropy_matches_the_definition(rows, vocabulary, width, dtype):
    _check(*_case(rows, vocabulary, width, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,vocabulary,width", [
    (2500, 6001, 136),
    (5200, 6001, 136),      # pairs of CTAs for the logits, single ones for the gradients
    (3001, 20003, 264),
    (5500, 35003, 264),     # pairs for both
    (200, 30000, 40),       # dH in slices of the vocabulary
    (200, 30000, 1100),     # logits in two segments of the features
    (2900, 20003, 517),
    (5500, 20003, 1029)])   # pairs, element-wise rows, segments
def test_linear_cross_entropy_every_kind_of_product(rows, vocabulary, width, dtype):
    hidden, weight, targets = _case(rows, vocabulary, width, dtype, ignored=0.1, seed=14)
    first = _check(hidden, weight, targets)
    second = _check(hidden, weight, targets)
    assert all(torch.equal(a, b) for a, b in zip(first, second)), "not the same bits twice"


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.98])
@pytest.mark.parametrize("scale", [1.0, -0.5])
def test_linear_cross_entropy_reductions_and_ignored_rows(reduction, ignored, scale, dtype):
    hidden, weight, targets = _case(300, 700, 96, dtype, ignored=ignored, seed=1)
    generator = torch.Generator(device="cuda").manual_seed(2)
    upstream = torch.randn(300, device="cuda", generator=generator) if reduction == "none" \
        else torch.tensor(0.125, device="cuda")
    _check(hidden, weight, targets, reduction=reduction, scale=scale, upstream=upstream)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy_every_row_ignored(reduction):
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(140, 300, 72, BF16)
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    loss = linear_cross_entropy(hidden, weight, torch.full_like(targets, -100), reduction=reduction)
    assert loss.isnan() if reduction == "mean" else not loss.any()
    for grad, leaf in zip(torch.autograd.grad(loss, leaves, torch.ones_like(loss)), leaves):
        assert grad.shape == leaf.shape and not grad.any()


def test_linear_cross_entropy_other_ignore_index_and_int32():
    hidden, weight, targets = _case(200, 300, 64, BF16)
    targets[::3] = 7
    _check(hidden, weight, targets.int(), ignore_index=7)


def test_linear_cross_entropy_ignored_rows_may_hold_anything():
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(300, 500, 136, BF16, ignored=0.4, seed=3)
    drop = targets == -100
    dirty = hidden.clone()
    dirty[drop] = torch.tensor(float("nan"), dtype=BF16, device="cuda")
    dirty[drop.nonzero()[0]] = torch.tensor(float("inf"), dtype=BF16, device="cuda")
    results = []
    for h in (hidden, dirty):
        leaves = [h.requires_grad_(), weight.requires_grad_()]
        loss = linear_cross_entropy(*leaves, targets)
        results.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not results[1][1][drop].any()


def test_linear_cross_entropy_targets_outside_the_vocabulary_are_not_numbers():
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(20, 50, 64, BF16)
    for wrong in (50, -1, 2**40, -2**62):
        bad = targets.clone()
        bad[3] = wrong
        losses = linear_cross_entropy(hidden, weight, bad, reduction="none")
        assert losses[3].isnan() and losses.isnan().sum() == 1
        leaves = [hidden.requires_grad_(), weight.requires_grad_()]
        loss = linear_cross_entropy(*leaves, bad)
        dhidden, dweight = torch.autograd.grad(loss, leaves)
        assert loss.isnan() and dhidden[3].isnan().all() and dweight.isnan().all()
        assert dhidden[:3].isfinite().all() and dhidden[4:].isfinite().all()


def test_linear_cross_entropy_large_logits():
    """Logits in the thousands: exp of them overflows, the losses do not."""
    hidden, weight, targets = _case(150, 400, 64, BF16, seed=4)
    _check(hidden, weight, targets, scale=1000.0, reduction="none")
    hidden, weight, targets = _case(150, 400, 64, FP16, seed=4)
    _check(hidden, weight, targets, scale=-300.0, reduction="sum")


@pytest.mark.parametrize("train", [False, True])
def test_linear_cross_entropy_small_losses_keep_their_digits(train):
    """A confident row: z = (a, 0, ..), exact in BF16, loss = log(1 + 6 exp(-a)).  The target's logit
    is the maximum, so what is rounded is a sum just over one (2^-23 at most) and its logarithm."""
    from attnres.loss import linear_cross_entropy
    for width in (16, 512):
        hidden = torch.zeros(40, width, device="cuda", dtype=BF16)
        hidden[:, 3] = torch.arange(40, device="cuda") / 2
        weight = torch.zeros(7, width, device="cuda", dtype=BF16)
        weight[5, 3] = 1
        targets = torch.full((40,), 5, device="cuda")
        weight.requires_grad_(train)
        want = torch.log1p(6 * torch.exp(-hidden[:, 3].double()))
        got = linear_cross_entropy(hidden, weight, targets, reduction="none").detach().double()
        assert ((got - want).abs() <= 2 * E * (1 + want)).all(), (got - want).abs().max()
        for row in (10, 20, 30):
            total = linear_cross_entropy(hidden[row:], weight, targets[row:], reduction="sum").item()
            assert abs(total - want[row:].sum().item()) <= (40 - row) * 2 * E * (1 + want[row].item())


def test_linear_cross_entropy_infinities_and_nan_in_a_row_that_counts():
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(10, 300, 64, BF16)
    hidden[2, 5], hidden[7, 1] = float("inf"), float("nan")
    losses = linear_cross_entropy(hidden, weight, targets, reduction="none")
    clean = [0, 1, 3, 4, 5, 6, 8, 9]
    assert losses[[2, 7]].isnan().all() and losses[clean].isfinite().all()
    assert torch.equal(losses[clean], linear_cross_entropy(hidden[clean], weight, targets[clean],
                                                           reduction="none"))


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_linear_cross_entropy_upstream_weights_of_any_size(dtype):
    """Weights far below and above what the inputs' type holds are carried in FP32."""
    hidden, weight, targets = _case(130, 300, 64, dtype, seed=5)
    for size in (1e-9, 1e-4, 1.0, 300.0):
        upstream = size * torch.rand(130, device="cuda", generator=torch.Generator(
            device="cuda").manual_seed(6))
        if dtype == FP16 and size < 1.0:   # gradients under FP16's range: only that they are finite
            from attnres.loss import linear_cross_entropy
            leaves = [hidden.requires_grad_(), weight.requires_grad_()]
            for grad in torch.autograd.grad(
                    linear_cross_entropy(*leaves, targets, reduction="none"), leaves, upstream):
                assert grad.isfinite().all()
        else:
            _check(hidden, weight, targets, reduction="none", upstream=upstream)
    zero = torch.zeros(130, device="cuda")
    assert not any(g.any() for g in _check(hidden, weight, targets, reduction="none", upstream=zero)[1:])


@pytest.mark.parametrize("width", [96, 640])
def test_linear_cross_entropy_upstream_of_one_number(width):
    hidden, weight, targets = _case(200, 300, width, BF16, ignored=0.2, seed=15)
    for upstream in (1.0, 0.3, -7.0, 0.0):
        _check(hidden, weight, targets, upstream=torch.tensor(upstream, device="cuda"))
    for upstream in (float("inf"), float("nan")):
        from attnres.loss import linear_cross_entropy
        loss = linear_cross_entropy(hidden, weight, targets)
        grads = torch.autograd.grad(loss, (hidden, weight), torch.tensor(upstream, device="cuda"))
        assert not any(g.isfinite().all() for g in grads)


@pytest.mark.parametrize("width", [96, 640])
def test_linear_cross_entropy_backward_twice_through_one_forward(width):
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(200, 300, width, BF16, ignored=0.2, seed=16)
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    loss = linear_cross_entropy(hidden, weight, targets)
    first = torch.autograd.grad(loss, leaves, torch.tensor(2.0, device="cuda"), retain_graph=True)
    second = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, 2 * b) for a, b in zip(first, second))


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_linear_cross_entropy_wide_rows_special_cases(reduction):
    """The cases above that are narrow, where the forward forms the gradients."""
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(140, 300, 520, BF16, seed=17)
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    loss = linear_cross_entropy(hidden, weight, torch.full_like(targets, -100), reduction=reduction)
    assert loss.isnan() if reduction == "mean" else not loss.any()
    assert not any(g.any() for g in torch.autograd.grad(loss, leaves))
    bad = targets.clone()
    bad[3] = 300
    loss = linear_cross_entropy(*leaves, bad, reduction=reduction)
    dhidden, dweight = torch.autograd.grad(loss, leaves)
    assert loss.isnan() and dhidden[3].isnan().all() and dweight.isnan().all()
    assert dhidden[:3].isfinite().all() and dhidden[4:].isfinite().all()
    drop = torch.arange(140, device="cuda") % 3 == 0
    masked = torch.where(drop, -100, targets)
    results = []
    for filler in (0.0, float("nan"), float("inf")):
        dirty = torch.where(drop[:, None], torch.tensor(filler, dtype=BF16, device="cuda"), hidden.detach())
        pair = [dirty.requires_grad_(), weight]
        loss = linear_cross_entropy(*pair, masked, reduction=reduction)
        results.append([loss.detach(), *torch.autograd.grad(loss, pair)])
    assert all(torch.equal(a, b) for other in results[1:] for a, b in zip(results[0], other))
    _check(hidden.detach(), weight.detach(), targets, reduction=reduction, scale=300.0)


def test_linear_cross_entropy_strange_upstream_weights_stay_with_their_rows():
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(30, 300, 64, BF16)
    upstream = torch.ones(30, device="cuda")
    upstream[4], upstream[9] = float("nan"), float("inf")
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    dhidden, dweight = torch.autograd.grad(
        linear_cross_entropy(*leaves, targets, reduction="none"), leaves, upstream)
    rest = [i for i in range(30) if i not in (4, 9)]
    assert dhidden[rest].isfinite().all() and not dhidden[[4, 9]].isfinite().any()
    assert dweight.isnan().any()


@pytest.mark.parametrize("rows,vocabulary,width,ignored", [
    (40000, 8200, 64, 0.0),
    (66000, 4999, 40, 0.2),
    (9000, 140000, 24, 0.2),     # logits in blocks of rows, three pieces of the vocabulary
    (70000, 8300, 40, 0.2),      # two pieces of the vocabulary, the last of them short
    (70000, 8300, 39, 0.0),
    (66500, 8300, 512, 0.1),     # gradients in the forward, two pieces of the rows
    (66500, 8301, 515, 0.0),
])
def test_linear_cross_entropy_in_pieces(rows, vocabulary, width, ignored):
    hidden, weight, targets = _case(rows, vocabulary, width, BF16, ignored=ignored, seed=7)
    first = _check(hidden, weight, targets)
    second = _check(hidden, weight, targets)
    assert all(torch.equal(a, b) for a, b in zip(first, second)), "not the same bits twice"


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,vocabulary,width", [
    (10, 30001, 520),       # dH in slices of the vocabulary, beside the logits and after them
    (3, 9000, 1030),
    (1900, 13, 40),         # too short to be cut
    (5201, 13, 40),         # dW in slices of the rows
    (5001, 130, 515),
    (2048, 9050, 77),       # more of dH than of dW
    (6500, 6400, 512),      # tiles for every SM: none
    (4600, 4500, 130),      # both
])
def test_linear_cross_entropy_gradients_in_slices(rows, vocabulary, width, dtype):
    hidden, weight, targets = _case(rows, vocabulary, width, dtype, ignored=0.1, seed=21)
    first = _check(hidden, weight, targets, reduction="sum")
    second = _check(hidden, weight, targets, reduction="sum")
    assert all(torch.equal(a, b) for a, b in zip(first, second)), "not the same bits twice"
    # a few kept rows leave most slices of dW empty, and none leaves them all so
    from attnres.loss import linear_cross_entropy
    targets[3:] = -100
    _check(hidden.detach(), weight.detach(), targets)
    loss = linear_cross_entropy(hidden, weight, torch.full_like(targets, -100), reduction="sum")
    dhidden, dweight = torch.autograd.grad(loss, (hidden, weight))
    assert loss == 0 and not dhidden.any() and not dweight.any()


@pytest.mark.parametrize("rows,vocabulary,width", [
    (1000, 600000, 512),    # two pieces of the rows, dH in slices in each
    (180000, 3000, 512),    # two pieces of the rows, dW in slices in each
])
def test_linear_cross_entropy_slices_in_pieces(rows, vocabulary, width):
    _check(*_case(rows, vocabulary, width, BF16, ignored=0.1, seed=22))


@pytest.mark.parametrize("needed", ["hidden", "weight"])
@pytest.mark.parametrize("rows,vocabulary,width", [(20, 9000, 520), (20, 9000, 72), (6000, 30, 520), (6000, 30, 72)])
def test_linear_cross_entropy_slices_of_the_gradient_that_is_wanted(needed, rows, vocabulary, width):
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(rows, vocabulary, width, BF16, seed=23)
    both = _check(hidden, weight, targets)
    hidden, weight = hidden.detach(), weight.detach()
    leaf = (hidden if needed == "hidden" else weight).requires_grad_()
    got, = torch.autograd.grad(linear_cross_entropy(hidden, weight, targets), leaf)
    assert torch.equal(got, both[1 if needed == "hidden" else 2])


@pytest.mark.parametrize("layout", ["one row", "three axes", "padded rows", "odd offset", "strided features",
                                    "expanded rows", "padded head", "transposed head", "odd head",
                                    "strided targets", "expanded upstream"])
def test_linear_cross_entropy_layouts(layout):
    hidden, weight, targets = _case(120, 260, 64, BF16, seed=8)
    options = {}
    wide = torch.randn(120, 200, device="cuda").to(BF16)
    head = (torch.randn(260, 200, device="cuda") / 8).to(BF16)
    if layout == "one row":
        hidden, targets = hidden[7], targets[7]
    elif layout == "three axes":
        hidden, targets = hidden.view(4, 30, 64), targets.view(4, 30)
    elif layout == "padded rows":
        hidden = wide[:, :64]
    elif layout == "odd offset":
        hidden = wide[:, 3:67]
    elif layout == "strided features":
        hidden = wide[:, 0:128:2]
    elif layout == "expanded rows":
        hidden = wide[:1, :64].expand(120, 64)
    elif layout == "padded head":
        weight = head[:, 8:72]
    elif layout == "transposed head":
        weight = (torch.randn(64, 260, device="cuda") / 8).to(BF16).t()
    elif layout == "odd head":
        weight = head[:, 5:69]
    elif layout == "strided targets":
        targets = torch.stack((targets, targets + 1), 1)[:, 0]
    else:
        options = dict(reduction="none", upstream=torch.full((1,), 0.5, device="cuda").expand(120))
    _check(hidden.detach(), weight.detach(), targets, **options)


def test_linear_cross_entropy_no_rows():
    from attnres.loss import linear_cross_entropy
    for reduction in ("mean", "sum", "none"):
        hidden = torch.empty(2, 0, 64, device="cuda", dtype=BF16, requires_grad=True)
        weight = torch.randn(30, 64, device="cuda").to(BF16).requires_grad_()
        loss = linear_cross_entropy(hidden, weight, torch.empty(2, 0, device="cuda", dtype=torch.int64),
                                    reduction=reduction)
        assert loss.shape == ((2, 0) if reduction == "none" else ())
        assert reduction == "none" or (loss.isnan() if reduction == "mean" else loss == 0)
        dhidden, dweight = torch.autograd.grad(loss, (hidden, weight), torch.ones_like(loss))
        assert dhidden.shape == hidden.shape and not dweight.any()


@pytest.mark.parametrize("needed", ["hidden", "weight"])
@pytest.mark.parametrize("width", [72, 512])
def test_linear_cross_entropy_only_the_gradient_that_is_wanted(needed, width):
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(150, 300, width, BF16, seed=9)
    both = _check(hidden, weight, targets)
    hidden, weight = hidden.detach(), weight.detach()
    leaf = (hidden if needed == "hidden" else weight).requires_grad_()
    got, = torch.autograd.grad(linear_cross_entropy(hidden, weight, targets), leaf)
    assert torch.equal(got, both[1 if needed == "hidden" else 2])


def test_linear_cross_entropy_gradient_against_differences():
    """The slope of the loss along a random direction against the gradient's component in it.  The
    direction's step is exact in BF16 (a power of two times +-1 on values that are multiples of
    it), so the only errors are the loss's (1e-5 / step) and curvature (step^2)."""
    from attnres.loss import linear_cross_entropy
    generator = torch.Generator(device="cuda").manual_seed(10)
    step = 2.0**-5
    grid = lambda *s: (torch.randint(-16, 17, s, device="cuda", generator=generator) * step)  # noqa: E731
    hidden, weight = grid(20, 32), grid(50, 32)
    targets = torch.randint(50, (20,), device="cuda", generator=generator)
    leaves = [hidden.to(BF16).requires_grad_(), weight.to(BF16).requires_grad_()]
    grads = torch.autograd.grad(linear_cross_entropy(*leaves, targets), leaves)
    for position in range(2):
        direction = torch.randint(0, 2, grads[position].shape, device="cuda", generator=generator) * 2.0 - 1.0
        ends = []
        for sign in (1, -1):
            moved = [hidden.clone(), weight.clone()]
            moved[position] += sign * step * direction
            assert torch.equal(moved[position].to(BF16).float(), moved[position])
            ends.append(linear_cross_entropy(*(m.to(BF16) for m in moved), targets).double())
        slope = ((ends[0] - ends[1]) / (2 * step)).item()
        along = (grads[position].double() * direction).sum().item()
        size = (grads[position].double().abs()).sum().item()
        assert abs(slope - along) < 2.0**-8 * size + 0.02, (slope, along)


@pytest.mark.parametrize("width", [64, 576])
def test_linear_cross_entropy_compiles_and_captures(width):
    from attnres.loss import linear_cross_entropy
    hidden, weight, targets = _case(160, 300, width, BF16, ignored=0.2, seed=11)
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    for reduction in ("mean", "none"):
        call = lambda h, w, t: linear_cross_entropy(h, w, t, reduction=reduction)  # noqa: E731
        loss = call(*leaves, targets)
        want = [loss.detach(), *torch.autograd.grad(loss, leaves, torch.ones_like(loss))]
        torch.compiler.reset()
        compiled = torch.compile(call, fullgraph=True)(*leaves, targets)
        got = [compiled.detach(), *torch.autograd.grad(compiled, leaves, torch.ones_like(compiled))]
        assert all(torch.equal(a, e) for a, e in zip(got, want))
    static = [t.detach().clone().requires_grad_() for t in leaves]
    ids = targets.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(linear_cross_entropy(*static, ids), static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(*static, ids)
        grads = torch.autograd.grad(loss, static)
    other = _case(160, 300, width, BF16, ignored=0.7, seed=12)   # another number of rows that count
    with torch.no_grad():
        for dst, src in zip((*static, ids), other):
            dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    again = [other[0].requires_grad_(), other[1].requires_grad_()]
    expected = linear_cross_entropy(*again, other[2])
    assert torch.equal(loss, expected)
    assert all(torch.equal(a, e) for a, e in zip(grads, torch.autograd.grad(expected, again)))


def test_linear_cross_entropy_writes_only_its_outputs():
    from attnres import _native
    pad = 64
    for rows, vocabulary, width in ((130, 300, 64), (67, 259, 37), (3, 5003, 41), (6001, 5, 72)):
        hidden, weight, targets = _case(rows, vocabulary, width, BF16, ignored=0.3, seed=13)
        padded = (width + 7) // 8 * 8

        def guarded(count, kind):
            whole = torch.full((count + 2 * pad,), -7, device="cuda", dtype=kind)
            return whole, whole[pad:pad + count]

        buffers = {}
        def take(name, count, kind):
            buffers[name], view = guarded(count, kind)
            return view.data_ptr()
        kept, index = take("kept", rows * padded, BF16), take("index", rows, torch.int32)
        target, count = take("target", rows, torch.int32), take("count", 1, torch.int32)
        sums, losses = take("sums", rows, FP32), take("losses", rows, FP32)
        loss, dh = take("loss", 1, FP32), take("dh", rows * width, BF16)
        dw = take("dw", vocabulary * width, BF16)
        size = _native.loss_workspace_bytes(rows, vocabulary, width, _native.LOSS_FORWARD)
        space = take("space", size // 4, FP32)
        stream = torch.cuda.current_stream().cuda_stream
        common = (targets.data_ptr(), 1, rows, vocabulary, width, 0, -100, 1.0, 2)
        _native.loss_forward(hidden.data_ptr(), width, weight.data_ptr(), width, *common, kept, index,
                             target, count, sums, losses, loss, None, None, space, size, stream)
        size = _native.loss_workspace_bytes(rows, vocabulary, width, _native.LOSS_BACKWARD)
        space = take("space back", size // 4, FP32)
        one = torch.ones(1, device="cuda")
        _native.loss_backward(one.data_ptr(), 1, weight.data_ptr(), width, *common, kept, index, target,
                              count, sums, dh, dw, space, size, stream)
        size = _native.loss_workspace_bytes(rows, vocabulary, width, _native.LOSS_FORWARD_GRADIENTS)
        space = take("space gradients", size // 4, FP32)
        dh, dw = take("dh early", rows * width, BF16), take("dw early", vocabulary * width, BF16)
        _native.loss_forward(hidden.data_ptr(), width, weight.data_ptr(), width, *common, kept, index,
                             target, count, None, losses, loss, dh, dw, space, size, stream)
        torch.cuda.synchronize()
        for name, whole in buffers.items():
            assert bool((whole[:pad] == -7).all()) and bool((whole[-pad:] == -7).all()), name


@pytest.mark.parametrize("width", [72, 520])
def test_linear_cross_entropy_on_two_streams_in_inference_mode_and_twice(width):
    """Two calls at once, each with its own workspace; and no second derivative."""
    from attnres.loss import linear_cross_entropy
    cases = [_case(700, 3000, width, BF16, ignored=0.2, seed=seed) for seed in (20, 21)]
    leaves = [[h.requires_grad_(), w.requires_grad_()] for h, w, _ in cases]
    call = lambda i: torch.autograd.grad(linear_cross_entropy(*leaves[i], cases[i][2]), leaves[i])  # noqa: E731
    want = [call(i) for i in range(2)]
    loss = linear_cross_entropy(*leaves[0], cases[0][2])
    with torch.inference_mode():
        assert torch.equal(linear_cross_entropy(*leaves[0], cases[0][2]), loss)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for g in got[i] for a, b in zip(g, want[i]))
    grads = torch.autograd.grad(loss, leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):
        grads[0].float().sum().backward()


def test_no_product_gave_up_waiting():
    from attnres import _native
    torch.cuda.synchronize()
    assert _native.error_flag() == 0
