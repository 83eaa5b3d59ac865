"""embed against its definition in 64 bits, forward and backward.

Tolerances: with u = 2^-24 and h half a step of the result's type, a result is rounded once to its
type after FP32 arithmetic: |out - out64| <= h |out| + 2 u (|s t| + |p|); a gradient that adds n
terms is off by at most h |d| + (n + 4) u sum|terms|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24


def _inside(got, want, slack, what):
    info = torch.finfo(got.dtype)
    off = (got.double() - want).abs()
    limit = info.eps / 2 * want.abs() + slack + info.smallest_normal * info.eps / 2
    assert got.shape == want.shape, what
    assert not (off > limit).any().item() and got.isfinite().all(), (what, off.max().item())


def _check(tokens, table, positions=None, *, scale=1.0, padding_idx=None, dtype=None, seed=0,
           upstream=None):
    from attnres.embedding import embed
    leaves = [t.requires_grad_() for t in (table, positions) if t is not None]
    out = embed(tokens, table, positions, scale=scale, padding_idx=padding_idx, dtype=dtype)
    assert out.dtype == (dtype or table.dtype) and out.shape == (*tokens.shape, table.shape[1])
    s64, ids = torch.tensor(scale, dtype=FP32).double().item(), tokens.long().reshape(-1)
    width, period = table.shape[1], tokens.shape[-1] if tokens.ndim else 1
    scaled = s64 * table.detach().double()[ids]
    added = torch.zeros(period, width, device="cuda", dtype=torch.float64) if positions is None \
        else positions.detach().double()
    added = added.repeat(ids.numel() // period, 1)
    _inside(out.detach().reshape(-1, width), scaled + added, 2 * U * (scaled.abs() + added.abs()), "out")
    if upstream is None:
        generator = torch.Generator(device="cuda").manual_seed(seed)
        upstream = torch.randn(out.shape, device="cuda", generator=generator).to(out.dtype)
    grads = torch.autograd.grad(out, leaves, upstream)
    g = s64 * upstream.double().reshape(-1, width)
    if padding_idx is not None:
        g = g * (ids != padding_idx % table.shape[0])[:, None]
    want = torch.zeros(table.shape, device="cuda", dtype=torch.float64).index_add_(0, ids, g)
    size = torch.zeros_like(want).index_add_(0, ids, g.abs())
    uses = torch.bincount(ids, minlength=table.shape[0])[:, None]
    _inside(grads[0], want, (uses + 4) * U * size, "dtable")
    if positions is not None:
        g = upstream.double().reshape(-1, period, width)
        _inside(grads[1], g.sum(0), (g.shape[0] + 4) * U * g.abs().sum(0), "dpositions")
    return out.detach(), grads


def _table(vocabulary, width, dtype, seed=1):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(vocabulary, width, device="cuda", generator=generator)).to(dtype)


def _ids(shape, vocabulary, seed=2, kind=torch.int64):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(vocabulary, shape, device="cuda", generator=generator).to(kind)


# widths from one column to the widest, odd ones (element accesses) and powers of two; vocabularies
# of one to three sort passes
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape,vocabulary,width", [
    ((1, 1), 1, 1), ((1, 1), 5, 8), ((2, 3), 2, 7), ((3, 33), 31, 16), ((2, 100), 257, 24),
    ((4, 65), 511, 31), ((1, 700), 512, 64), ((5, 129), 1000, 200), ((2, 1024), 32000, 96),
    ((3, 17), 70000, 40), ((1, 50), 300000, 8), ((2, 31), 50, 1001), ((2, 40), 97, 1024),
    ((1, 9), 11, 4096), ((1, 5), 7, 8191), ((2, 3), 7, 8192)])
def test_embed_matches_the_definition(shape, vocabulary, width, dtype):
    _check(_ids(shape, vocabulary), _table(vocabulary, width, dtype),
           _table(shape[-1], width, dtype, 3), scale=0.7, seed=4)


@pytest.mark.parametrize("table,positions,out", [
    (FP32, FP32, BF16), (BF16, FP32, FP16), (FP16, BF16, FP32), (FP32, None, FP16), (BF16, None, BF16)])
@pytest.mark.parametrize("kind", [torch.int64, torch.int32], ids=["int64", "int32"])
def test_embed_types(table, positions, out, kind):
    _check(_ids((3, 50), 90, kind=kind), _table(90, 72, table),
           None if positions is None else _table(50, 72, positions, 3), dtype=out, scale=math.sqrt(72))


@pytest.mark.parametrize("width", [40, 37, 1024])
@pytest.mark.parametrize("pattern", ["one id", "two ids", "sorted", "reversed", "all distinct",
                                     "zipf", "last id only", "runs of 32", "runs of 33"])
def test_embed_gradient_for_every_distribution(pattern, width):
    """Runs of equal ids inside a tile of sorted tokens, across two, across many."""
    n, vocabulary = 3000, 4000
    i = torch.arange(n, device="cuda")
    tokens = {"one id": torch.full_like(i, 17), "two ids": i % 2 * 3999, "sorted": i,
              "reversed": n - 1 - i, "all distinct": (i * 1237) % vocabulary,
              "zipf": (1.0 / (torch.rand(n, device="cuda", generator=torch.Generator(
                  device="cuda").manual_seed(5)) + 1e-3)).long().clamp_(0, 3999),
              "last id only": torch.full_like(i, 3999), "runs of 32": i // 32,
              "runs of 33": i // 33}[pattern]
    _, first = _check(tokens[None], _table(vocabulary, width, FP32), seed=6)
    _, second = _check(tokens[None], _table(vocabulary, width, FP32), seed=6)
    assert torch.equal(first[0], second[0]), "not the same bits twice"


def test_embed_gradient_is_summed_in_token_order():
    """Terms whose FP32 sum depends on the order: 1, then many 2^-24 (each lost), then -1."""
    from attnres.embedding import embed
    n = 31
    table = torch.zeros(4, 8, device="cuda", requires_grad=True)
    tokens = torch.full((1, n), 2, device="cuda")
    upstream = torch.full((1, n, 8), 2.0**-24, device="cuda")
    upstream[0, 0], upstream[0, n - 1] = 1.0, -1.0
    grad, = torch.autograd.grad(embed(tokens, table), table, upstream)
    assert not grad[2].any() and not grad[[0, 1, 3]].any()


@pytest.mark.parametrize("kind", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("width", [16, 37, 264, 1001, 2056])
@pytest.mark.parametrize("n", [1, 31, 33, 127, 128, 129, 256])
def test_embed_few_tokens(n, width, kind):
    """Up to 128 tokens are not sorted."""
    for vocabulary, ids in ((9, torch.full((n,), 8)), (5, torch.arange(n) * 7 % 5),
                            (40000, 39999 - torch.arange(n)), (300, torch.arange(n) * n % 300)):
        for padding_idx in (None, int(ids[n // 2])):
            _, first = _check(ids.cuda()[None], _table(vocabulary, width, kind), _table(n, width, FP32, 3),
                              scale=0.6, padding_idx=padding_idx, seed=n)
            _, second = _check(ids.cuda()[None], _table(vocabulary, width, kind),
                               _table(n, width, FP32, 3), scale=0.6, padding_idx=padding_idx, seed=n)
            assert all(torch.equal(a, b) for a, b in zip(first, second)), "not the same bits twice"


def test_embed_few_tokens_in_the_order_of_more():
    """The sums are those of a sorted call where no run crosses a tile of 32."""
    from attnres.embedding import embed
    ids = torch.arange(120, device="cuda") * 17 % 47
    upstream = _table(120, 72, FP32, 9)
    grads = []
    for extra in (0, 100):   # the others have no gradient
        table = _table(47, 72, FP32).requires_grad_()
        tokens = torch.cat((ids, torch.full((extra,), 1 << 20, device="cuda")))
        more = torch.cat((upstream, upstream[:extra]))
        grads.append(torch.autograd.grad(embed(tokens[None], table), table, more[None])[0])
    assert torch.allclose(grads[0], grads[1], rtol=4 * U, atol=4 * U * 3 * upstream.abs().max().item())


@pytest.mark.parametrize("n", [32, 33, 4096, 131073, 200000])
def test_embed_many_tokens(n):
    """Past 131 072 tokens the tiles grow; the sort's shares are longer than a warp."""
    _check(_ids((1, n), 5000, 7), _table(5000, 16, FP32), seed=8)


@pytest.mark.parametrize("n,vocabulary,width,dtype,positions", [
    (3000, 60000, 512, FP32, False), (3000, 60000, 513, BF16, True), (16384, 30000, 1024, FP32, True),
    (1, 100000, 520, FP32, False), (40, 2000000, 24, FP32, False)])
def test_embed_large_tables(n, vocabulary, width, dtype, positions):
    """Tables whose zero rows take longer to write than the ids to sort: the first rows are written
    beside the sort, the rest beside the sums; ids at both ends of both parts."""
    tokens = _ids((1, n), vocabulary, 10)
    if n > 3:
        tokens[0, :3] = torch.tensor([0, vocabulary - 1, vocabulary // 3])
    _check(tokens, _table(vocabulary, width, dtype), _table(n, width, dtype, 3) if positions else None)


@pytest.mark.parametrize("padding_idx", [0, 5, -1])
def test_embed_padding_row_gets_no_gradient(padding_idx):
    tokens = _ids((4, 90), 10)
    _, grads = _check(tokens, _table(10, 48, BF16), padding_idx=padding_idx, scale=2.0)
    assert not grads[0][padding_idx].any() and grads[0].any()


def test_embed_padding_only():
    _, grads = _check(torch.full((2, 40), 3, device="cuda"), _table(10, 48, FP32), padding_idx=3)
    assert not grads[0].any()


def test_embed_ids_outside_the_table():
    """Nothing is read or written out of range; the row says so and gets no gradient."""
    from attnres.embedding import embed
    table, positions = _table(10, 64, FP32).requires_grad_(), _table(5, 64, FP32).requires_grad_()
    tokens = torch.tensor([[0, -1, 10, 2**40, 9], [-2**63, 3, 3, 2**31, 2**32 + 1]], device="cuda")
    out = embed(tokens, table, positions)
    bad = (tokens < 0) | (tokens >= 10)
    assert out[bad].isnan().all() and out[~bad].isfinite().all()
    upstream = torch.ones_like(out)
    dtable, dpositions = torch.autograd.grad(out, (table, positions), upstream)
    want = torch.zeros_like(table).index_add_(0, tokens[~bad], upstream[~bad])
    assert torch.equal(dtable, want) and torch.equal(dpositions, torch.full_like(positions, 2.0))


def test_embed_masked_gradients_stay_with_their_id():
    """An infinity in one token's gradient reaches that id's row and no other."""
    from attnres.embedding import embed
    table = _table(50, 40, FP32).requires_grad_()
    tokens = _ids((1, 400), 50)
    upstream = torch.randn(1, 400, 40, device="cuda")
    upstream[0, 123] = float("inf")
    grad, = torch.autograd.grad(embed(tokens, table), table, upstream)
    hit = tokens[0, 123]
    assert grad[hit].isinf().all()
    grad[hit] = 0
    assert grad.isfinite().all()


@pytest.mark.parametrize("layout", ["padded table", "odd table", "transposed table", "strided ids",
                                    "scalar ids", "no batch axis", "sliced gradient", "expanded gradient"])
def test_embed_layouts(layout):
    tokens, table, positions, upstream = _ids((4, 30), 60), _table(60, 64, FP32), None, None
    if layout == "padded table":
        table = _table(60, 80, FP32)[:, :64]
    elif layout == "odd table":
        table = _table(60, 81, BF16)[:, 3:67]
    elif layout == "transposed table":
        table = _table(64, 60, FP32).t()
    elif layout == "strided ids":
        tokens = _ids((30, 8), 60)[:, ::2].t()
    elif layout == "scalar ids":
        tokens, positions = _ids((), 60), _table(1, 64, FP32)
    elif layout == "no batch axis":
        tokens, positions = _ids((30,), 60), _table(40, 64, FP32)[:30]
    elif layout == "sliced gradient":
        upstream = torch.randn(4, 30, 72, device="cuda")[..., 4:68]
    else:
        upstream = torch.ones((), device="cuda").expand(4, 30, 64)
    _check(tokens, table, positions, upstream=upstream)


@pytest.mark.parametrize("n", [100, 400])
@pytest.mark.parametrize("layout", ["odd table", "transposed table", "strided ids", "sliced gradient",
                                    "odd gradient", "expanded gradient"])
def test_embed_layouts_sorted_and_not(layout, n):
    tokens, table, positions, upstream = _ids((2, n // 2), 60), _table(60, 64, FP32), None, None
    if layout == "odd table":
        table = _table(60, 81, BF16)[:, 3:67]
    elif layout == "transposed table":
        table, positions = _table(64, 60, FP32).t(), _table(64, n // 2, FP32).t()
    elif layout == "strided ids":
        tokens = _ids((n // 2, 8), 60)[:, ::4].t()
    elif layout == "sliced gradient":
        upstream = torch.randn(2, n // 2, 72, device="cuda")[..., 4:68]
    elif layout == "odd gradient":
        upstream = torch.randn(2, n // 2, 67, device="cuda")[..., 3:]
    else:
        upstream = torch.ones((), device="cuda").expand(2, n // 2, 64)
    _check(tokens, table, positions, upstream=upstream)


@pytest.mark.parametrize("n", [90, 500])
def test_embed_bad_ids_padding_and_infinities_sorted_and_not(n):
    from attnres.embedding import embed
    torch.manual_seed(3)
    table = _table(50, 40, FP32).requires_grad_()
    _, grads = _check(torch.full((2, n // 2), 3, device="cuda"), table.detach(), padding_idx=3)
    assert not grads[0].any()
    tokens, upstream = _ids((n,), 50), torch.randn(n, 40, device="cuda")
    strange = torch.tensor([-1, 50, 2**40, -2**63, 2**31, 2**32 + 1, -2**31], device="cuda")
    where = torch.randperm(n, device="cuda")[:7]
    tokens[where] = strange
    upstream[where] = float("nan")      # of rows without an id: reaches nothing
    upstream[where[0] - 1] = float("inf")
    hit = tokens[where[0] - 1]
    grad, = torch.autograd.grad(embed(tokens, table), table, upstream)
    fine = (tokens >= 0) & (tokens < 50) & (tokens != hit)
    want = torch.zeros(50, 40, device="cuda", dtype=torch.float64)
    want.index_add_(0, tokens[fine], upstream[fine].double())
    size = torch.zeros_like(want).index_add_(0, tokens[fine], upstream[fine].abs().double())
    if 0 <= int(hit) < 50:
        assert grad[hit].isinf().all()
        grad[hit] = 0
    _inside(grad, want, (n + 4) * U * size, "dtable")


@pytest.mark.parametrize("needed", ["table", "positions"])
def test_embed_only_the_gradient_that_is_wanted_sorted(needed):
    from attnres.embedding import embed
    tokens, table, positions = _ids((3, 140), 70), _table(70, 24, FP32), _table(140, 24, FP32, 3)
    leaf = (table if needed == "table" else positions).requires_grad_()
    out = embed(tokens, table, positions)
    got, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    want = torch.bincount(tokens.reshape(-1), minlength=70)[:, None].expand(70, 24) \
        if needed == "table" else torch.full((140, 24), 3.0, device="cuda")
    assert torch.equal(got, want.float())


def test_embed_few_tokens_captured():
    from attnres.embedding import embed
    table = _table(500, 264, BF16).requires_grad_()
    ids, upstream = _ids((1, 40), 500), _table(40, 264, BF16, 5)[None]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(embed(ids, table), table, upstream)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad, = torch.autograd.grad(embed(ids, table), table, upstream)
    ids.copy_(_ids((1, 40), 500, 9))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, torch.autograd.grad(embed(ids, table), table, upstream)[0])


def test_embed_no_tokens():
    from attnres.embedding import embed
    table, positions = _table(10, 16, BF16).requires_grad_(), _table(5, 16, BF16).requires_grad_()
    out = embed(torch.empty(0, 5, device="cuda", dtype=torch.int64), table, positions)
    assert out.shape == (0, 5, 16)
    for grad, leaf in zip(torch.autograd.grad(out, (table, positions), torch.empty_like(out)),
                          (table, positions)):
        assert grad.shape == leaf.shape and not grad.any()


@pytest.mark.parametrize("needed", ["table", "positions"])
def test_embed_only_the_gradient_that_is_wanted(needed):
    from attnres.embedding import embed
    tokens, table, positions = _ids((3, 40), 70), _table(70, 24, FP32), _table(40, 24, FP32, 3)
    leaf = (table if needed == "table" else positions).requires_grad_()
    out = embed(tokens, table, positions)
    got, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    want = torch.bincount(tokens.reshape(-1), minlength=70)[:, None].expand(70, 24) \
        if needed == "table" else torch.full((40, 24), 3.0, device="cuda")
    assert torch.equal(got, want.float())


def test_embed_compiles_and_captures():
    from attnres.embedding import embed
    tokens, table, positions = _ids((4, 64), 100), _table(100, 96, FP32), _table(64, 96, FP32, 3)
    leaves = [table.requires_grad_(), positions.requires_grad_()]
    call = lambda t, a, b: embed(t, a, b, scale=2.0, padding_idx=1, dtype=BF16)  # noqa: E731
    upstream = torch.randn(4, 64, 96, device="cuda").to(BF16)
    out = call(tokens, *leaves)
    want = [out.detach(), *torch.autograd.grad(out, leaves, upstream)]
    compiled = torch.compile(call, fullgraph=True)(tokens, *leaves)
    got = [compiled.detach(), *torch.autograd.grad(compiled, leaves, upstream)]
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    static = [t.detach().clone().requires_grad_() for t in leaves]
    ids = tokens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(call(ids, *static), static, upstream)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(ids, *static)
        grads = torch.autograd.grad(out, static, upstream)
    ids.copy_(_ids((4, 64), 100, 9))
    graph.replay()
    torch.cuda.synchronize()
    expected = call(ids, *leaves)
    assert torch.equal(out, expected)
    assert all(torch.equal(a, e) for a, e in zip(grads, torch.autograd.grad(expected, leaves, upstream)))


def test_embed_writes_only_its_outputs():
    from attnres import _native
    period, vocabulary, pad = 100, 77, 64
    for n, width, code, dtype in ((300, 64, 2, FP32), (300, 37, 0, BF16), (300, 1030, 1, FP16),
                                  (100, 64, 0, BF16), (100, 1030, 2, FP32)):
        tokens, table = _ids((n,), vocabulary), _table(vocabulary, width, dtype)

        def guarded(count, kind):
            whole = torch.full((count + 2 * pad,), -7, device="cuda", dtype=kind)
            return whole, whole[pad:pad + count]

        out_all, out = guarded(n * width, dtype)
        dt_all, dtable = guarded(vocabulary * width, dtype)
        dp_all, dpos = guarded(period * width, FP32)
        size = _native.embedding_workspace_bytes(n, width)
        ws_all, workspace = guarded(size // 4, FP32)
        assert size % 4 == 0
        stream = torch.cuda.current_stream().cuda_stream
        _native.embedding_forward(tokens.data_ptr(), 1, n, period, vocabulary, width, table.data_ptr(),
                                  width, code, None, 0, 2, 1.0, out.data_ptr(), code, stream)
        _native.embedding_backward(tokens.data_ptr(), 1, n, period, vocabulary, width, -1,
                                   out.data_ptr(), width, code, 1.0, dtable.data_ptr(), code,
                                   dpos.data_ptr(), 2, workspace.data_ptr(), size, stream)
        torch.cuda.synchronize()
        for whole in (out_all, dt_all, dp_all, ws_all):
            assert bool((whole[:pad] == -7).all()) and bool((whole[-pad:] == -7).all())
        assert torch.equal(out.view(n, width), table[tokens])


def test_embed_on_two_streams_in_inference_mode_and_twice():
    """Two gradients at once, each with its own workspace; and no second derivative."""
    from attnres.embedding import embed
    tables = [_table(3000, 264, FP32, seed).requires_grad_() for seed in (1, 2)]
    tokens = [_ids((4, 700), 3000, seed) for seed in (3, 4)]
    upstream = torch.randn(4, 700, 264, device="cuda")
    want = [torch.autograd.grad(embed(t, w), w, upstream)[0] for t, w in zip(tokens, tables)]
    with torch.inference_mode():
        assert torch.equal(embed(tokens[0], tables[0]), tables[0][tokens[0]])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(torch.autograd.grad(embed(tokens[i], tables[i]), tables[i], upstream)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    grad, = torch.autograd.grad(embed(tokens[0], tables[0]).sum(), tables[0], create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
