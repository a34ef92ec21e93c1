"""Low-rank adapters of many requests: forward, gradients and refusals against the definition in 64 bits.

Tolerances are derived: the sums over K and the rank run in f32 (an error of at most (K + rank + 16) 2^-24 of the sum of the terms' sizes),
the hidden vector enters the second product as two bf16 parts (2^-17 of it, three parts 2^-25 for an f32 result), and a result is rounded once
to its type, by at most half a step (bf16: 2^-8 of the value)."""

import itertools

import pytest
import torch

import wave_b200 as wb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def make(rows, K, N, rank, pool, y_dtype=BF16, ids="mixed", seed=0, scale=True, id_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, y = r(rows, K).to(BF16), r(rows, N).to(y_dtype)
    a, b = (r(pool, rank, K) * K ** -0.5).to(BF16), (r(pool, N, rank) * 0.3).to(BF16)
    s = torch.rand(pool, generator=g) + 0.5 if scale else None
    if ids == "mixed":
        at = torch.randint(-1, pool, (rows,), generator=g)
    elif ids == "runs":
        at = torch.sort(torch.randint(0, pool, (rows,), generator=g)).values
    elif ids == "none":
        at = torch.full((rows,), -1)
    else:
        at = torch.full((rows,), pool - 1)
    return [t.to(DEV) if t is not None else None for t in (y, x, a, b, at.to(id_dtype), s)]


def definition(y, x, a, b, ids, s, g=None):
    """(out, sizes) in 64 bits, sizes being the sums of the terms' absolute values; with g also the gradients of x, a and b, each with sizes."""
    y, x, a, b = (t.detach().double() for t in (y, x, a, b))
    ids = ids.long()
    out, size = y.clone(), torch.zeros_like(y)
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    sx, sa, sb = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for l in range(a.shape[0]):  # noqa: E741
        at = (ids == l).nonzero()[:, 0]
        f = float(s[l].double()) if s is not None else 1.0
        h, hs = x[at] @ a[l].T, x[at].abs() @ a[l].abs().T
        out[at] += f * (h @ b[l].T)
        size[at] = f * (hs @ b[l].abs().T)
        if g is not None:
            gl = g[at].double()
            u, us = f * (gl @ b[l]), f * (gl.abs() @ b[l].abs())
            dx[at], sx[at] = u @ a[l], us @ a[l].abs()
            da[l], sa[l] = u.T @ x[at], us.T @ x[at].abs()
            db[l], sb[l] = f * (gl.T @ h), f * (gl.abs().T @ hs)
    return ((out, size), (dx, sx), (da, sa), (db, sb)) if g is not None else (out, size)


def assert_near(got, want, size, terms, parts):
    """parts: of the hidden vector; terms: of the longest sums."""
    assert got.shape == want.shape
    tol = size * (2.0 ** (-17 if parts == 2 else -25) + (terms + 16) * 2.0 ** -24)
    tol = tol + (want.abs() + tol) * (2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24) + 1e-38
    over = (got.double() - want).abs() - tol
    assert bool((over <= 0).all()), f"{int((over > 0).sum())} of {over.numel()} off, by {float(over.max())}"


def check_forward(args, **kw):
    y, x, a, b, ids, s = args
    got = wb.apply_adapters(y, x, a, b, ids, s, **kw)
    want, size = definition(y, x, a, b, ids, s)
    assert got.dtype == y.dtype
    assert_near(got, want, size, x.shape[1] + a.shape[1], 2 if y.dtype == BF16 else 3)
    untouched = (ids < 0) | (ids >= a.shape[0])
    assert torch.equal(got[untouched], y[untouched])
    return got


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 33, 64, 65, 130, 600])
@pytest.mark.parametrize("rank,pool", [(1, 3), (8, 1), (16, 70), (20, 5), (64, 9)])
def test_forward_rows_and_ranks(rows, rank, pool):
    check_forward(make(rows, 256, 200, rank, pool, seed=rows * rank))


@pytest.mark.parametrize("K,N", [(8, 1), (32, 7), (264, 33), (1024, 4001), (4096, 64), (2048, 1030), (96, 1096)])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("rank", [7, 12, 64, 100, 256])
def test_forward_widths_and_types(K, N, y_dtype, rank):
    check_forward(make(90, K, N, rank, 4, y_dtype, ids="runs", seed=K + N))
    check_forward(make(5, K, N, rank, 4, y_dtype, ids="mixed", seed=K + N + 1))


@pytest.mark.parametrize("ids", ["mixed", "runs", "none", "last"])
@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
def test_forward_ids(ids, id_dtype):
    check_forward(make(200, 512, 300, 16, 33, ids=ids, id_dtype=id_dtype, scale=False))


def test_ids_outside_the_pool_have_no_adapter():
    args = make(70, 128, 96, 8, 4, id_dtype=torch.int64)
    args[4][::3] = 2 ** 40
    args[4][1::3] = -(2 ** 40)
    check_forward(args)


def test_in_place_and_given_output():
    args = make(150, 256, 130, 16, 5)
    want = check_forward(args)
    out = torch.empty_like(args[0])
    assert wb.apply_adapters(*args, out=out) is out and torch.equal(out, want)
    y = args[0].clone()
    assert wb.apply_adapters(y, *args[1:], out=y) is y and torch.equal(y, want)


def test_strided_rows():
    """Column blocks of wider matrices, odd pitches, rows that are no multiple of 16 bytes apart, a transposed pool."""
    y, x, a, b, ids, s = make(77, 256, 100, 16, 5)
    want = check_forward([y, x, a, b, ids, s])
    for pad_x, pad_y in ((8, 4), (3, 1), (1, 27)):
        wide_x, wide_y = torch.full((77, 256 + pad_x), float("nan"), dtype=BF16, device=DEV), torch.full((77, 100 + pad_y), float("nan"), dtype=BF16, device=DEV)
        wide_x[:, pad_x:], wide_y[:, :100] = x, y
        assert torch.equal(wb.apply_adapters(wide_y[:, :100], wide_x[:, pad_x:], a, b, ids, s), want)
        out = torch.zeros(77, 100 + pad_y, dtype=BF16, device=DEV)
        wb.apply_adapters(y, x, a, b, ids, s, out=out[:, pad_y:])
        assert torch.equal(out[:, pad_y:], want) and not out[:, :pad_y].any()
    assert torch.equal(wb.apply_adapters(y.T.contiguous().T, x, a.transpose(1, 2).contiguous().transpose(1, 2), b, ids, s), want)
    expanded = wb.apply_adapters(y[:1].expand(77, 100), x[:1].expand(77, 256), a, b, ids, s)
    assert torch.equal(expanded, wb.apply_adapters(y[:1].repeat(77, 1), x[:1].repeat(77, 1), a, b, ids, s))


def test_values_that_are_not_finite_stay_in_their_rows():
    y, x, a, b, ids, s = make(100, 256, 96, 16, 4)
    want = wb.apply_adapters(y, x, a, b, ids, s)
    ids[10], ids[20], ids[30] = 1, 2, -1
    x2, y2 = x.clone(), y.clone()
    x2[10, 5], x2[20, 7], x2[30] = float("nan"), float("inf"), float("nan")
    y2[40, 3] = float("-inf")
    got = wb.apply_adapters(y2, x2, a, b, ids, s)
    clean = torch.ones(100, dtype=torch.bool, device=DEV)
    clean[[10, 20, 30, 40]] = False
    assert torch.equal(got[clean], want[clean])
    assert got[10].isnan().all() and torch.equal(got[30], y2[30])
    ref, _ = definition(y2, x2, a, b, ids, s)
    assert torch.equal(got[20].float().isinf(), ref[20].isinf()) and float(got[40, 3]) == float("-inf")


@pytest.mark.parametrize("rows,K,N,rank,pool,ids", [(1, 64, 64, 4, 1, "last"), (16, 256, 200, 8, 3, "mixed"), (130, 520, 333, 16, 4, "runs"), (300, 256, 1000, 32, 5, "mixed"),
                                                    (700, 1024, 512, 64, 2, "runs"), (260, 128, 264, 100, 3, "mixed"), (129, 2048, 96, 12, 30, "mixed"),
                                                    (64, 96, 65, 16, 7, "none"), (2000, 256, 256, 16, 1, "last"),
                                                    (500, 128, 1027, 20, 3, "mixed"), (40, 64, 1030, 8, 20, "mixed"), (5000, 64, 40, 4, 2, "mixed")])
def test_gradients(rows, K, N, rank, pool, ids):
    y, x, a, b, at, s = make(rows, K, N, rank, pool, ids=ids, seed=rows)
    g = (torch.randn(rows, N, generator=torch.Generator().manual_seed(1)) * 0.01).to(BF16).to(DEV)
    leaves = [t.clone().requires_grad_() for t in (y, x, a, b)]
    out = wb.apply_adapters(*leaves, at, s)
    grads = torch.autograd.grad(out, leaves, g)
    (want, size), (dx, sx), (da, sa), (db, sb) = definition(y, x, a, b, at, s, g)
    assert_near(out.detach(), want, size, K + rank, 2)
    assert torch.equal(grads[0], g)
    assert_near(grads[1], dx, sx, N + rank, 2)
    assert_near(grads[2], da, sa, N + rows, 2)
    assert_near(grads[3], db, sb, K + rows, 2)
    unused = ~torch.isin(torch.arange(pool, device=DEV), at)
    assert not grads[2][unused].any() and not grads[3][unused].any()
    again = torch.autograd.grad(wb.apply_adapters(*leaves, at, s), leaves, g)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # the same bits on every run
    assert all(torch.equal(_only(y, (x, a, b), i, at, s, g), grads[1 + i]) for i in range(3))


def _only(y, leaves, i, ids, s, g):
    """The gradient of one leaf where the others want none."""
    leaves = [t.clone().requires_grad_(i == j) for j, t in enumerate(leaves)]
    return torch.autograd.grad(wb.apply_adapters(y, *leaves, ids, s), leaves[i], g)[0]


def test_gradients_against_differences():
    """Central differences of the definition, in 64 bits, along random directions: within the roundings of the gradients (2^-8 of each, added up
    like independent errors: 8 standard deviations)."""
    y, x, a, b, ids, s = make(40, 64, 48, 8, 3)
    g = torch.randn(40, 48, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(wb.apply_adapters(y, *leaves, ids, s), leaves, g)
    for i, (leaf, grad) in enumerate(zip((x, a, b), grads)):
        d = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(DEV)
        f = [(definition(y, *[t.double() + (e * d if j == i else 0) for j, t in enumerate((x, a, b))], ids, s)[0] * g.double()).sum() for e in (1e-4, -1e-4)]
        want, got = (f[0] - f[1]) / 2e-4, (grad.double() * d).sum()
        assert abs(float(want - got)) <= 8 * 2.0 ** -8 * float((grad.double() * d).norm()) + 1e-6


def test_gradient_of_strided_and_expanded_tensors():
    y, x, a, b, ids, s = make(90, 128, 72, 16, 3)
    g = torch.randn(90, 72, generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
    want = [_only(y, (x, a, b), i, ids, s, g) for i in range(3)]
    wide = torch.zeros(90, 200, dtype=BF16, device=DEV)
    wide[:, 5:133] = x
    wide.requires_grad_()
    got, = torch.autograd.grad(wb.apply_adapters(y, wide[:, 5:133], a, b, ids, s), wide, g)
    assert torch.equal(got[:, 5:133], want[0]) and not got[:, :5].any()
    one = torch.randn(1, 72, generator=torch.Generator().manual_seed(5)).to(BF16).to(DEV)
    got = _only(y, (x, a, b), 1, ids, s, one.expand(90, 72))  # a gradient that is broadcast, as of a sum
    assert torch.equal(got, _only(y, (x, a, b), 1, ids, s, one.repeat(90, 1)))
    shared = x[:1].clone().requires_grad_()  # one row for all: its gradient is the sum over the rows
    got, = torch.autograd.grad(wb.apply_adapters(y, shared.expand(90, 128), a, b, ids, s), shared, g)
    rows = _only(y, (x[:1].repeat(90, 1), a, b), 0, ids, s, g)
    assert torch.allclose(got.float(), rows.float().sum(0, keepdim=True), rtol=2 ** -7, atol=1e-4)


# ---- the kernels on the tensor cores: many rows, ranks above 32 ------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,K,N,rank,pool,ids", [
    (2048, 512, 136, 8, 3, "runs"), (2500, 1024, 72, 16, 70, "mixed"), (2049, 64, 264, 24, 4, "mixed"), (300, 4096, 200, 64, 2, "runs"), (257, 192, 96, 100, 5, "mixed"),
    (70, 2048, 64, 256, 1, "last"), (4100, 1088, 64, 36, 2, "none"), (129, 64, 8, 40, 130, "mixed")])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
def test_many_rows_onto_the_ranks(rows, K, N, rank, pool, ids, y_dtype):
    check_forward(make(rows, K, N, rank, pool, y_dtype, ids, seed=rows))


@pytest.mark.parametrize("rows,K,N,rank,pool,ids", [
    (8192, 64, 4096, 64, 1, "last"), (8200, 128, 4104, 64, 7, "runs"), (65540, 64, 520, 40, 3, "mixed"), (4097, 64, 8264, 48, 130, "mixed"), (9000, 64, 3800, 56, 2, "none"),
    (131100, 64, 264, 64, 4, "runs")])
def test_many_rows_onto_the_columns(rows, K, N, rank, pool, ids):
    args = make(rows, K, N, rank, pool, ids=ids, seed=rows)
    got = check_forward(args)
    y = args[0].clone()  # in place, and beside other columns
    assert torch.equal(wb.apply_adapters(y, *args[1:], out=y), got)
    wide = torch.full((rows, N + 16), 7.0, dtype=BF16, device=DEV)
    wb.apply_adapters(*args, out=wide[:, 8:N + 8])
    assert torch.equal(wide[:, 8:N + 8], got) and bool((wide[:, :8] == 7).all()) and bool((wide[:, N + 8:] == 7).all())


@pytest.mark.parametrize("rows,K,N,rank,pool,ids", [(8200, 4160, 64, 64, 3, "runs"), (8500, 4000, 128, 48, 5, "mixed"), (2100, 256, 192, 16, 2, "runs"), (300, 64, 1024, 40, 3, "mixed")])
def test_gradients_of_many_rows(rows, K, N, rank, pool, ids):
    y, x, a, b, at, s = make(rows, K, N, rank, pool, ids=ids, seed=rows)
    g = torch.randn(rows, N, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    x, a, b = (t.requires_grad_() for t in (x, a, b))
    grads = torch.autograd.grad(wb.apply_adapters(y, x, a, b, at, s), (x, a, b), g)
    _, (dx, sx), (da, sa), (db, sb) = definition(y, x, a, b, at, s, g)
    for got, want, size, terms in zip(grads, (dx, da, db), (sx, sa, sb), (N + rank, rows + N, rows + K)):
        assert_near(got, want, size, terms, 2)


def test_an_adapter_that_is_not_finite_stays_with_its_rows():
    y, x, a, b, ids, s = make(8200, 64, 4096, 64, 5, ids="runs")
    want = wb.apply_adapters(y, x, a, b, ids, s)
    a, b = a.clone(), b.clone()
    a[1], b[3] = float("inf"), float("nan")
    x2 = x.clone()
    x2[5] = float("nan")
    got = wb.apply_adapters(y, x2, a, b, ids, s)
    clean = (ids != 1) & (ids != 3)
    clean[5] = False
    assert torch.equal(got[clean], want[clean]) and got[ids == 3].isnan().all() and got[5].isnan().all()


@pytest.mark.parametrize("rows,rank", [(2, 5), (40, 8), (150, 5), (150, 40)])
def test_an_infinity_meets_the_ranks_there_are(rows, rank):
    """Ranks are padded to sixteen: what an infinity of x would be in a rank that is not there (a NaN) does not reach the output."""
    y, x, a, b, ids, s = make(rows, 64, 48, rank, 3)
    ids[1] = 2
    x[1, 9] = float("inf")
    a[2] = a[2].abs() + 1
    b[2] = b[2].abs() + 1
    got = wb.apply_adapters(y, x, a, b, ids, s)
    assert (got[1] == float("inf")).all() and got[0].isfinite().all()


@pytest.mark.parametrize("rows", [3, 150])
def test_captured_and_replayed(rows):
    """Forward and backward in one graph, replayed on new inputs; two graphs of the same call do not disturb one another."""
    args = make(rows, 256, 200, 16, 5)
    y, x, a, b, ids, s = args
    g = torch.randn(rows, 200, generator=torch.Generator().manual_seed(6)).to(BF16).to(DEV)
    x, a, b = (t.requires_grad_() for t in (x, a, b))

    def step():
        out = wb.apply_adapters(y, x, a, b, ids, s)
        return [out.detach(), *torch.autograd.grad(out, (x, a, b), g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        graphs.append((graph, res))
    for seed in (7, 8):
        new = make(rows, 256, 200, 16, 5, seed=seed)
        with torch.no_grad():
            for old, fresh in zip((y, x, a, b, ids, s), new):
                old.copy_(fresh)
        want = step()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(p, q) for p, q in zip(res, want))


def test_other_stream():
    args = make(300, 512, 256, 16, 4)
    want = check_forward(args)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = [wb.apply_adapters(*args) for _ in range(5)]
    st.synchronize()
    assert all(torch.equal(t, want) for t in got)


def test_no_rows():
    y, x, a, b, ids, s = make(4, 64, 32, 8, 2)
    assert wb.apply_adapters(y[:0], x[:0], a, b, ids[:0], s).shape == (0, 32)
    a = a.requires_grad_()
    out = wb.apply_adapters(y[:0], x[:0], a, b, ids[:0], s)
    assert not torch.autograd.grad(out.sum(), a)[0].any()


def test_refusals():
    y, x, a, b, ids, s = make(8, 64, 32, 8, 3)
    apply = wb.apply_adapters
    bad = [(y, x.float(), a, b, ids, s), (y, x, a.half(), b, ids, s), (y.half(), x, a, b, ids, s), (y, x, a, b, ids.float(), s), (y, x, a, b, ids[:7], s),
           (y[:7], x, a, b, ids, s), (y, x[:, :56], a, b, ids, s), (y, x, a, b[:2], ids, s), (y, x, a, b[:, :31], ids, s), (y, x, a, b, ids, s[:2]),
           (y, x, a, b, ids, s.double()), (y, x, a, b, ids.cpu(), s), (y, x, a.cpu(), b, ids, s), (y, x[:, :60], a[:, :, :60], b, ids, s),
           (y, x, a[0], b, ids, s), (y, x, a[:, :0], b[:, :, :0], ids, s), (y, x, a[:0], b[:0], ids, s[:0])]
    for args in bad:
        with pytest.raises(ValueError):
            apply(*args)
    for out in (torch.empty(8, 32, device=DEV), torch.empty(8, 33, dtype=BF16, device=DEV), torch.empty(32, 8, dtype=BF16, device=DEV).T,
                torch.empty(8, 32, dtype=BF16)):
        with pytest.raises(ValueError):
            apply(y, x, a, b, ids, s, out=out)
    big = torch.zeros(1, 257, 64, dtype=BF16, device=DEV)
    with pytest.raises(ValueError):
        apply(y, x, big, torch.zeros(1, 32, 257, dtype=BF16, device=DEV), ids)
    x = x.requires_grad_()
    with pytest.raises(ValueError):
        apply(y, x, a, b, ids, s, out=y)
    with pytest.raises(ValueError):
        apply(y.float(), x, a, b, ids, s)
    with pytest.raises(ValueError):
        apply(y, x, a[:, :, :8].repeat(22000, 1, 1)[:, :1].repeat(1, 1, 8), b.repeat(22000, 1, 1)[:, :, :1], ids)
    with pytest.raises(ValueError):
        apply(y, x, a, b, ids, s.requires_grad_())


# ---- on the layer ---------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("shape", [(3,), (2, 5), (4, 70)])
def test_layer_with_adapters(shape):
    """The layer's output with the adapters on top, in place of the layer's own tensor; x of any leading shape."""
    g = torch.Generator().manual_seed(3)
    layer = wb.MXFP4Linear.from_float(torch.randn(192, 256, generator=g).to(DEV))
    pool = wb.LowRankAdapters(*[t.to(DEV) for t in ((torch.randn(4, 8, 256, generator=g) / 16).to(BF16), torch.randn(4, 192, 8, generator=g).to(BF16))])
    x = torch.randn(*shape, 256, generator=g).to(BF16).to(DEV)
    ids = torch.randint(-1, 4, shape, generator=g).to(DEV)
    plain = layer(x)
    got = layer(x, pool, ids)
    want = wb.apply_adapters(plain.reshape(-1, 192), x.reshape(-1, 256), pool.a, pool.b, ids.reshape(-1)).reshape(plain.shape)
    assert got.shape == (*shape, 192) and torch.equal(got, want)
    assert torch.equal(layer(x), plain)
    with pytest.raises(ValueError):
        layer(x, pool)
    with pytest.raises(ValueError):
        layer(x, pool, ids.reshape(-1)[:-1])
    with pytest.raises(ValueError):
        layer(x.float(), pool, ids)
    with pytest.raises(ValueError):  # the layer's part of the gradient would be missing
        layer(x.clone().requires_grad_(), pool, ids)


@pytest.mark.parametrize("trainable", [False, True])
@pytest.mark.parametrize("through", [False, True])
def test_layer_refuses_an_empty_batch_with_adapters_as_without(trainable, through):
    g = torch.Generator().manual_seed(3)
    layer = wb.MXFP4Linear.from_float(torch.randn(192, 256, generator=g).to(DEV), input_grad=True)
    pool = wb.LowRankAdapters(torch.zeros(4, 8, 256, dtype=BF16, device=DEV), torch.zeros(4, 192, 8, dtype=BF16, device=DEV), trainable=trainable)
    x = torch.zeros(0, 256, dtype=BF16, device=DEV, requires_grad=through)
    for args in ((x,), (x, pool, torch.zeros(0, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            layer(*args)


def test_layer_trains_adapters_through_frozen_layers():
    """Two layers with adapters, one behind the other: the gradients against those of the same network in 64 bits, whose activations are rounded
    as the layers round them (the rounding counts as the identity)."""
    g = torch.Generator().manual_seed(9)
    rows, sizes = 96, (256, 320, 128)
    layers = [wb.MXFP4Linear.from_float((torch.randn(n, k, generator=g) * k ** -0.5).to(DEV), input_grad=True) for k, n in zip(sizes, sizes[1:])]
    pools = [wb.LowRankAdapters((torch.randn(3, 8, k, generator=g) * k ** -0.5).to(BF16).to(DEV), (torch.randn(3, n, 8, generator=g) * 0.3).to(BF16).to(DEV),
                                torch.tensor([0.5, 1.0, 2.0], device=DEV), trainable=True) for k, n in zip(sizes, sizes[1:])]
    x = torch.randn(rows, sizes[0], generator=g).to(BF16).to(DEV).requires_grad_()
    ids = torch.randint(-1, 3, (rows,), generator=g).to(DEV)
    up = torch.randn(rows, sizes[-1], generator=g).to(BF16).to(DEV)
    mid = layers[0](x, pools[0], ids)
    out = layers[1](mid, pools[1], ids)
    leaves = [x, *[p for pool in pools for p in (pool.a, pool.b)]]
    grads = torch.autograd.grad(out, leaves, up)
    # by hand: each layer's backward from its own input, in 64 bits
    h, want = up, []
    for layer, pool, inp in reversed(list(zip(layers, pools, (x.detach(), mid.detach())))):
        w = wb.ops.dequant_mxfp4(layer.weight_codes, layer.weight_scales).double()
        _, (dx, _), (da, _), (db, _) = definition(torch.zeros(rows, w.shape[0], device=DEV), inp, pool.a, pool.b, ids, pool.scale, h)
        want = [da, db] + want
        h = h.double() @ w + dx
    for got, ref in zip(grads, [h] + want):
        # a relative error of 2^-8 enters at each of the roundings on the way (out of each layer's two parts, their sum, the result)
        assert float((got.double() - ref).norm()) <= 4 * 2.0 ** -8 * float(ref.norm())


@pytest.mark.parametrize("rows,N", [(5, 192), (200, 96), (90, 77)])
def test_layer_gradient_is_the_layers_part_with_the_adapters_on_it(rows, N):
    g = torch.Generator().manual_seed(rows)
    layer = wb.MXFP4Linear.from_float((torch.randn(N, 256, generator=g) / 16).to(DEV), input_grad=True)
    y, x, a, b, ids, s = make(rows, 256, N, 16, 4, seed=rows)
    pool = wb.LowRankAdapters(a, b, s)
    up = torch.randn(rows, N, generator=g).to(BF16).to(DEV)
    x.requires_grad_()
    out = layer(x, pool, ids)
    dx, = torch.autograd.grad(out, x, up)
    assert torch.equal(out.detach(), wb.apply_adapters(layer._base(x.detach()), x.detach(), a, b, ids, s))
    part = wb.mxfp4_input_grad(up, layer.weight_codes, layer.weight_scales)
    _, (want, size), _, _ = definition(y, x, a, b, ids, s, up)
    assert_near(dx, part.double() + want, size, N + 16, 2)
    assert torch.equal(dx[ids < 0], part[ids < 0])
    assert torch.equal(out.detach()[ids < 0], layer._base(x.detach())[ids < 0])


@pytest.mark.parametrize("ids", ["runs", "mixed"])
def test_layer_gradient_of_many_rows(ids):
    """The adapters' part added to the layer's in place by the kernels for many rows, whole chunks without an adapter among them."""
    rows, K, N = 8300, 4096, 96
    g = torch.Generator().manual_seed(4)
    layer = wb.MXFP4Linear.from_float((torch.randn(N, K, generator=g) / 64).to(DEV), input_grad=True)
    y, x, a, b, at, s = make(rows, K, N, 48, 4, ids=ids, seed=rows)
    at[1000:1500] = -1
    up = torch.randn(rows, N, generator=g).to(BF16).to(DEV)
    x.requires_grad_()
    dx, = torch.autograd.grad(layer(x, wb.LowRankAdapters(a, b, s), at), x, up)
    part = wb.mxfp4_input_grad(up, layer.weight_codes, layer.weight_scales)
    _, (want, size), _, _ = definition(y, x, a, b, at, s, up)
    assert_near(dx, part.double() + want, size, N + 48, 2)
    assert torch.equal(dx[at < 0], part[at < 0])


def test_every_combination_of_wanted_gradients():
    y, x, a, b, ids, s = make(70, 128, 64, 16, 3)
    g = torch.randn(70, 64, generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
    full = [t.clone().requires_grad_() for t in (y, x, a, b)]
    want = torch.autograd.grad(wb.apply_adapters(*full, ids, s), full, g)
    for mask in itertools.product((False, True), repeat=4):
        if not any(mask):
            continue
        leaves = [t.clone().requires_grad_(m) for t, m in zip((y, x, a, b), mask)]
        out = wb.apply_adapters(*leaves, ids, s)
        got = torch.autograd.grad(out, [t for t, m in zip(leaves, mask) if m], g)
        assert all(torch.equal(p, q) for p, q in zip(got, [w for w, m in zip(want, mask) if m]))
