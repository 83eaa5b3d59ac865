"""layer_norm against its definition in 64 bits, forward and backward.

Tolerances: u = 2^-24 is half a step of FP32, h half a step of the result's type.  A row's mean is
off by a few u max|x|, the centred values and rstd by as much relative to their sizes, so
  |y - y64|   <= h |y| + 32 u (|w| rstd max|x| + |y| + |b|)
  |dx - dx64| <= h |dx| + 64 u rstd (1 + rstd max|x|) (|gw| + mean|gw| + (|xh| + 1) (mean|gw xh| + mean|gw|))
  |dw - dw64| <= h |dw| + (n + 32) u sum |g| (|xh| + rstd max|x|)      (n additions in FP32 at most)
plus half the smallest subnormal of the type where that is what rounding leaves.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _inside(got, want, slack, what):
    assert got.dtype.is_floating_point and got.shape == want.shape, what
    off = (got.double() - want).abs()
    limit = _half(got.dtype) * want.abs() + slack + _floor(got.dtype)
    worst = (off - limit).max().item() if off.numel() else -1.0
    assert worst <= 0.0, (what, off.max().item(), worst)


def _reference(x, w, b, eps, g):
    """Everything in 64 bits, with the sizes the tolerances are made of."""
    x, g = x.double(), g.double()
    rows, width = x.shape
    w64 = torch.ones(width, device=x.device, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rstd
    y = xh * w64 + b64
    gw = g * w64
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    big = rstd * x.abs().amax(-1, keepdim=True)
    slack = dict(
        y=32 * U * (w64.abs() * big + y.abs() + b64.abs()),
        dx=64 * U * rstd * (1 + big) * (gw.abs() + gw.abs().mean(-1, keepdim=True) + (xh.abs() + 1) * (
            (gw * xh).abs().mean(-1, keepdim=True) + gw.abs().mean(-1, keepdim=True))),
        dw=(rows + 32) * U * (g.abs() * (xh.abs() + big)).sum(0),
        db=(rows + 32) * U * g.abs().sum(0))
    return dict(y=y, dx=dx, dw=(g * xh).sum(0), db=g.sum(0)), slack


def _check(x, w, b, g, eps=1e-5):
    from attnres.norm import layer_norm
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and y.is_contiguous()
    width = x.shape[-1]
    want, slack = _reference(x.detach().reshape(-1, width), w, b, eps, g.reshape(-1, width))
    _inside(y.detach().reshape(-1, width), want["y"], slack["y"], "y")
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None],
                     torch.autograd.grad(y, leaves, g)))
    for name, got in grads.items():
        _inside(got.reshape(-1, width) if name == "dx" else got, want[name], slack[name], name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)
    return y, grads


def _case(rows, width, dtype, seed, params=FP32, centre=0.4):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=generator)
    return ((1.5 * normal(rows, width) + centre).to(dtype), (1 + 0.1 * normal(width)).to(params),
            (0.1 * normal(width)).to(params), normal(rows, width).to(dtype))


# every instance: widths around each group size, odd ones (element accesses) and multiples of the
# 16-byte chunk, a single column, the widest
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,width", [
    (1, 1), (5, 2), (3, 7), (37, 8), (64, 255), (33, 256), (9, 257), (40, 260), (21, 512), (7, 777),
    (50, 1024), (11, 1025), (13, 2048), (6, 3001), (5, 4096), (4, 4097), (3, 4104), (2, 8191), (3, 8192)])
def test_layer_norm_matches_the_definition(rows, width, dtype):
    x, w, b, g = _case(rows, width, dtype, rows * 10007 + width)
    _check(x, w, b, g)


@pytest.mark.parametrize("params", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("which", ["both", "weight", "bias", "none"])
def test_layer_norm_parameters(params, which):
    x, w, b, g = _case(130, 384, BF16, 5, params)
    _check(x, w if which in ("both", "weight") else None, b if which in ("both", "bias") else None, g)


def test_layer_norm_mixed_parameter_types():
    x, w, b, g = _case(130, 384, FP16, 6)
    y, grads = _check(x, w.to(BF16).detach(), b, g)
    assert grads["dw"].dtype == BF16 and grads["db"].dtype == FP32


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,width", [(9001, 1024), (5003, 200), (1203, 4096), (611, 8192)])
def test_layer_norm_more_rows_than_one_pass_of_the_grid(rows, width, dtype):
    x, w, b, g = _case(rows, width, dtype, 7)
    _, first = _check(x, w, b, g)
    _, second = _check(x, w, b, g)
    assert all(torch.equal(first[k], second[k]) for k in first), "not the same bits twice"


def test_layer_norm_of_one_row_without_a_batch_axis_in_inference_mode_and_on_another_stream():
    from attnres.norm import layer_norm
    x, w, b, g = _case(1, 777, BF16, 16)
    _check(x[0], w, b, g[0])
    want = layer_norm(x, w, b).detach()
    with torch.inference_mode():
        assert torch.equal(layer_norm(x, w, b), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        results = [layer_norm(x, w, b).detach() for _ in range(20)]
    mine = [layer_norm(x, w, b).detach() for _ in range(20)]   # at the same time, on this one
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results + mine)


@pytest.mark.parametrize("layout", ["padded", "odd offset", "transposed", "every other", "expanded",
                                    "three axes", "swapped axes"])
def test_layer_norm_layouts(layout):
    x, w, b, g = _case(60, 128, FP32, 8)
    wide = torch.randn(60, 300, device="cuda")
    if layout == "padded":
        x = wide[:, :128]
    elif layout == "odd offset":
        x, g = wide[:, 3:131], torch.randn(60, 300, device="cuda")[:, 1:129]
    elif layout == "transposed":
        x, g = torch.randn(128, 60, device="cuda").t(), torch.randn(128, 60, device="cuda").t()
    elif layout == "every other":
        x = wide[:, 0:256:2]
    elif layout == "expanded":
        x, g = torch.randn(1, 128, device="cuda").expand(60, 128), torch.ones((), device="cuda").expand(60, 128)
        return _check_expanded(x, w, b, g)
    elif layout == "three axes":
        x, g = x.view(4, 15, 128), g.view(4, 15, 128)
    else:
        x, g = torch.randn(15, 4, 128, device="cuda").transpose(0, 1), g.view(4, 15, 128)
    _check(x, w, b, g)


def _check_expanded(x, w, b, g):
    from attnres.norm import layer_norm
    leaf = x[:1].clone().requires_grad_()
    y = layer_norm(leaf.expand(60, 128), w, b)
    want, slack = _reference(x, w, b, 1e-5, g)
    _inside(y.detach(), want["y"], slack["y"], "y")
    got = torch.autograd.grad(y, leaf, g)[0]
    _inside(got[0], want["dx"].sum(0), (slack["dx"] + 64 * U * want["dx"].abs()).sum(0), "dx")


def test_layer_norm_large_mean_keeps_its_precision():
    """A mean 4000 times the spread: the sum of centred squares loses nothing."""
    x, w, b, g = _case(40, 1000, FP32, 9, centre=6000.0)
    _check(x, w, b, g)


def test_layer_norm_rows_of_constants_infinities_and_nan():
    from attnres.norm import layer_norm
    x, w, b, g = _case(6, 512, BF16, 10)
    x[1] = 3.0                                    # variance zero
    x[3, 100] = float("inf")
    x[4, 7] = float("nan")
    y = layer_norm(x, w, b)
    assert torch.equal(y[1], b.to(BF16))
    assert y[3].isnan().any() and y[4].isnan().all()
    clean = torch.tensor([0, 1, 2, 5], device="cuda")
    assert y[clean].isfinite().all()
    assert torch.equal(y[clean], layer_norm(x[clean], w, b)), "a row depends on its neighbours"
    zero = layer_norm(torch.full((2, 64), 5.0, device="cuda"), eps=0.0)
    assert zero.isnan().all()                     # 0 / 0, as the definition has it


def test_layer_norm_no_rows():
    from attnres.norm import layer_norm
    x = torch.empty(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == (0, 64)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 64, device="cuda", dtype=BF16))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


@pytest.mark.parametrize("needed", ["x", "weight", "bias", "x weight"])
def test_layer_norm_only_the_gradients_that_are_wanted(needed):
    from attnres.norm import layer_norm
    x, w, b, g = _case(77, 640, BF16, 11)
    named = dict(x=x, weight=w, bias=b)
    leaves = [named[n].requires_grad_() for n in needed.split()]
    got = torch.autograd.grad(layer_norm(x, w, b), leaves, g)
    want, slack = _reference(x.detach(), w.detach(), b.detach(), 1e-5, g)
    key = dict(x="dx", weight="dw", bias="db")
    for n, grad in zip(needed.split(), got):
        _inside(grad, want[key[n]], slack[key[n]], n)


def test_layer_norm_gradient_against_differences():
    """Central differences of a scalar of the output, in FP32 with a step that balances rounding
    (u |f| / step) and curvature (step^2): both under 2e-3 of the gradient's size here."""
    from attnres.norm import layer_norm
    generator = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(2, 24, device="cuda", generator=generator)
    w = 1 + 0.3 * torch.randn(24, device="cuda", generator=generator)
    b = torch.zeros(24, device="cuda")
    g = torch.randn(2, 24, device="cuda", generator=generator)
    f = lambda x, w, b: (layer_norm(x, w, b).double() * g.double()).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    step = 2.0**-7
    for position, grad in enumerate(grads):
        for index in range(0, grad.numel(), 5):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in (x, w, b)]
                moved[position].view(-1)[index] += sign * step
                ends.append(f(*moved))
            slope = ((ends[0] - ends[1]) / (2 * step)).item()
            assert abs(slope - grad.view(-1)[index].item()) < 2e-3 * (1 + grad.abs().max().item())


def test_layer_norm_compiles_and_captures():
    from attnres.norm import layer_norm
    x, w, b, g = _case(64, 512, BF16, 13)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    want = [layer_norm(x, w, b).detach(), *torch.autograd.grad(layer_norm(x, w, b), leaves, g)]
    compiled = torch.compile(layer_norm, fullgraph=True)
    y = compiled(x, w, b)
    assert all(torch.equal(a, e) for a, e in zip([y.detach(), *torch.autograd.grad(y, leaves, g)], want))

    static = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    upstream = g.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(layer_norm(*static), static, upstream)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(*static)
        grads = torch.autograd.grad(y, static, upstream)
    x2, _, _, g2 = _case(64, 512, BF16, 14)
    with torch.no_grad():
        static[0].copy_(x2)
    upstream.copy_(g2)
    graph.replay()
    torch.cuda.synchronize()
    again = [x2.requires_grad_(), *leaves[1:]]
    expected = layer_norm(*again)
    assert torch.equal(y, expected)
    assert all(torch.equal(a, e) for a, e in zip(grads, torch.autograd.grad(expected, again, g2)))


def test_layer_norm_double_backward_is_refused():
    from attnres.norm import layer_norm
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    grad, = torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_layer_norm_writes_only_its_outputs():
    """Raw calls with guard bands around every output."""
    from attnres import _native
    for rows, width, code, dtype in ((37, 1024, 0, BF16), (19, 333, 2, FP32), (5, 4100, 1, FP16)):
        x, w, b, g = _case(rows, width, dtype, 15)
        pad = 64

        def guarded(count, kind):
            whole = torch.full((count + 2 * pad,), -7, device="cuda", dtype=kind)
            return whole, whole[pad:pad + count]

        y_all, y = guarded(rows * width, dtype)
        s_all, stats = guarded(2 * rows, FP32)
        dx_all, dx = guarded(rows * width, dtype)
        dw_all, dw = guarded(width, FP32)
        db_all, db = guarded(width, FP32)
        stream = torch.cuda.current_stream().cuda_stream
        _native.norm_forward(x.data_ptr(), width, w.data_ptr(), b.data_ptr(), rows, width, code, 2,
                             1e-5, y.data_ptr(), stats.data_ptr(), stream)
        count = _native.norm_workspace_rows(rows, width, 0)
        p_all, partials = guarded(count * 2 * width, FP32)
        _native.norm_backward(g.data_ptr(), width, x.data_ptr(), width, stats.data_ptr(), w.data_ptr(),
                              rows, width, code, 2, dx.data_ptr(), partials.data_ptr(), count,
                              dw.data_ptr(), db.data_ptr(), stream)
        torch.cuda.synchronize()
        for whole in (y_all, s_all, dx_all, dw_all, db_all, p_all):
            assert bool((whole[:pad] == -7).all()) and bool((whole[-pad:] == -7).all())
        want, slack = _reference(x, w, b, 1e-5, g)
        _inside(y.view(rows, width), want["y"], slack["y"], "y")
        _inside(dx.view(rows, width), want["dx"], slack["dx"], "dx")
        _inside(dw, want["dw"], slack["dw"], "dw")
        _inside(db, want["db"], slack["db"], "db")
