"""Router, balance loss and the gradient of the weighted combine, against their definitions in 64 bits.

Tolerances: softmax and its gradient in f32 with the library's expf (2 units in the last place) and sums of E terms: a relative 2^-24 (E + 32) of the
terms; sums over the rows 2^-24 (rows / 8 + 64); bf16 results are rounded once (2^-8)."""

import pytest
import torch

import wave_b200 as wb
from wave_b200 import moe, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def make(rows, E, dtype=F32, seed=0, padded=False):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, E, generator=g) * 2).to(dtype).to(DEV)
    return logits, ((torch.rand(rows, generator=g) < 0.7).to(DEV) if padded else None)


def choose(z, k):
    """The k largest of every row, the lower index first among equals, NaN above all; on the host, from the definition."""
    rows = []
    for row in z.float().cpu().tolist():
        order = sorted(range(len(row)), key=lambda e: (0 if row[e] != row[e] else 1, -row[e] if row[e] == row[e] else 0.0, e))
        rows.append(order[:k])
    return torch.tensor(rows, dtype=torch.int64, device=DEV).reshape(len(rows), k)


def definition(logits, k, mask, renormalize, ids=None):
    """(weight, ids, counts, loss), differentiable, in 64 bits."""
    z = logits.double()
    rows, E = z.shape
    valid = torch.ones(rows, dtype=torch.bool, device=DEV) if mask is None else mask
    chosen = choose(logits.detach(), k) if ids is None else ids.long()
    p = torch.softmax(z, 1)
    inside = (chosen >= 0) & (chosen < E) & valid[:, None]
    weight = torch.gather(p, 1, chosen.clamp(0, E - 1))
    if renormalize:
        weight = weight / weight.sum(1, keepdim=True)
    weight = torch.where(valid[:, None], weight, 0.0)
    counts = torch.bincount(chosen[inside], minlength=E)
    n = max(1, int(valid.sum()))
    loss = E * (counts.double() / (chosen.shape[1] * n) * torch.where(valid[:, None], p, 0.0).sum(0) / n).sum()
    return weight, torch.where(valid[:, None], chosen, -1), counts, loss


def near(got, want, rel):
    assert got.shape == want.shape
    tol = want.abs() * rel + 1e-36
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / (want.abs() + 1e-30)).max())


@pytest.mark.parametrize("rows", [1, 7, 8, 64, 65, 500, 3001])
@pytest.mark.parametrize("E,k", [(1, 1), (8, 2), (31, 5), (33, 8), (100, 32), (256, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward(rows, E, k, dtype):
    logits, mask = make(rows, E, dtype, seed=rows + E, padded=rows % 2 == 1)
    for renormalize in (False, True):
        r = wb.router(logits, k, mask, renormalize)
        weight, ids, counts, loss = definition(logits, k, mask, renormalize)
        assert r.ids.dtype == torch.int32 and torch.equal(r.ids.long(), ids)
        assert r.counts.dtype == torch.int32 and torch.equal(r.counts.long(), counts)
        near(r.weight, weight, (E + 32) * 2.0 ** -24)
        near(r.balance_loss, loss, (E + rows / 8 + 96) * 2.0 ** -24)
        again = wb.router(logits, k, mask, renormalize)
        assert torch.equal(again.weight, r.weight) and torch.equal(again.balance_loss, r.balance_loss)


@pytest.mark.parametrize("rows,E,k", [(1, 2, 1), (16, 8, 2), (100, 40, 4), (700, 256, 8), (65, 64, 32)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("padded", [False, True])
def test_gradient(rows, E, k, dtype, renormalize, padded):
    logits, mask = make(rows, E, dtype, seed=rows, padded=padded)
    logits.requires_grad_()
    g = torch.Generator().manual_seed(1)
    gw, gl = torch.randn(rows, k, generator=g).to(DEV), torch.tensor(3.7, device=DEV)
    for use in ("both", "weight", "loss"):
        r = wb.router(logits, k, mask, renormalize)
        weight, _, _, loss = definition(logits, k, mask, renormalize)
        got = want = 0.0
        if use != "loss":
            got, want = got + (r.weight * gw).sum(), want + (weight * gw.double()).sum()
        if use != "weight":
            got, want = got + r.balance_loss * gl, want + loss * gl.double()
        dz, = torch.autograd.grad(got, logits)
        z64 = logits.detach().double().requires_grad_()
        weight, _, _, loss = definition(z64, k, mask, renormalize, ids=choose(logits.detach(), k))
        want = ((weight * gw.double()).sum() if use != "loss" else 0.0) + (loss * gl.double() if use != "weight" else 0.0)
        ref, = torch.autograd.grad(want, z64)
        # p (dp - sum p dp): the terms are at most 2 max|dp| p; with renormalize dp is divided by the chosen p's sum
        p = torch.softmax(z64.detach(), 1)
        wide = p if not renormalize else p / torch.gather(p, 1, choose(logits.detach(), k)).sum(1, keepdim=True)
        size = 4 * wide * (gw.double().abs().max() if use != "loss" else 0.0) * k + 4 * p * (3.7 * E if use != "weight" else 0.0) / max(1, rows if mask is None else int(mask.sum()))
        tol = size * (E + 64) * 2.0 ** -24 + ref.abs() * (2.0 ** -8 if dtype == BF16 else 2.0 ** -23) + 1e-36
        assert dz.dtype == dtype and bool(((dz.double() - ref).abs() <= tol).all())
        if mask is not None:
            assert not dz[~mask].any()


def test_gradient_against_differences():
    logits, mask = make(20, 12, padded=True)
    logits.requires_grad_()
    g = torch.randn(20, 3, generator=torch.Generator().manual_seed(2)).to(DEV)
    ids = choose(logits.detach(), 3)
    for renormalize in (False, True):
        r = wb.router(logits, 3, mask, renormalize)
        dz, = torch.autograd.grad((r.weight * g).sum() + r.balance_loss, logits)
        d = torch.randn(20, 12, generator=torch.Generator().manual_seed(3), dtype=torch.float64).to(DEV)
        f = []
        for e in (1e-5, -1e-5):
            weight, _, _, loss = definition(logits.detach().double() + e * d, 3, mask, renormalize, ids)
            f.append((weight * g.double()).sum() + loss)
        want, got = float((f[0] - f[1]) / 2e-5), float((dz.double() * d).sum())
        assert abs(want - got) <= 1e-5 * float((dz.double() * d).abs().sum()) + 1e-8


def test_ties_infinities_and_nan():
    inf, nan = float("inf"), float("nan")
    rows = [[1.0, 1.0, 1.0, 1.0, 1.0], [0.0, -0.0, 0.0, -0.0, -1.0], [-inf, 2.0, -inf, 1.0, -inf], [-inf] * 4 + [3.0],
            [torch.finfo(F32).min] * 5, [1.0, nan, 2.0, nan, 3.0]]
    for dtype in (F32, BF16):
        rows[4] = [torch.finfo(dtype).min] * 5  # the lowest finite value; f32's would be bf16's -inf, and a row of -inf has no softmax
        logits = torch.tensor(rows, device=DEV).to(dtype)
        r = wb.router(logits, 3)
        assert r.ids.tolist() == [[0, 1, 2], [0, 1, 2], [1, 3, 0], [4, 0, 1], [0, 1, 2], [1, 3, 4]]
        assert torch.allclose(r.weight[:5], torch.gather(torch.softmax(logits[:5].float(), 1), 1, r.ids[:5].long()), rtol=1e-6)
        assert r.weight[5].isnan().all() and r.balance_loss.isnan()
        mask = torch.tensor([True] * 5 + [False], device=DEV)  # a NaN behind the mask spoils nothing
        r = wb.router(logits, 3, mask)
        _, _, counts, loss = definition(logits[:5], 3, None, False)
        assert torch.equal(r.counts.long(), counts) and abs(float(r.balance_loss) - float(loss)) <= 1e-5 * float(loss)
        z = logits.clone().requires_grad_()
        r = wb.router(z, 3, mask, renormalize=True)
        dz, = torch.autograd.grad(r.weight.square().sum() + r.balance_loss, z)
        assert dz.isfinite().all() and not dz[5].any()


def test_masks_that_leave_nothing():
    for rows in (5, 300):
        logits, _ = make(rows, 16)
        logits.requires_grad_()
        r = wb.router(logits, 2, torch.zeros(rows, dtype=torch.bool, device=DEV))
        assert not r.weight.any() and bool((r.ids == -1).all()) and not r.counts.any() and float(r.balance_loss.detach()) == 0.0
        assert not torch.autograd.grad(r.balance_loss + r.weight.sum(), logits)[0].any()
    r = wb.router(logits[:0], 2)
    assert r.weight.shape == (0, 2) and r.ids.shape == (0, 2) and not r.counts.any() and float(r.balance_loss.detach()) == 0.0


@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,E,k", [(5, 6, 2), (400, 60, 40), (9, 256, 1)])
def test_balance_loss_of_given_choices(rows, E, k, id_dtype):
    """Repeated and out-of-range ids among them."""
    logits, mask = make(rows, E, padded=True)
    ids = torch.randint(-1, E + 2, (rows, k), generator=torch.Generator().manual_seed(4)).to(id_dtype).to(DEV)
    if id_dtype == torch.int64:
        ids[0, 0] = 2 ** 33
    logits.requires_grad_()
    for m in (None, mask):
        loss, counts = wb.balance_loss(logits, ids, m)
        z64 = logits.detach().double().requires_grad_()
        _, _, want_counts, want = definition(z64, k, m, False, ids=ids)
        assert torch.equal(counts.long(), want_counts)
        near(loss.detach(), want.detach(), (E + rows / 8 + 96) * 2.0 ** -24)
        dz, = torch.autograd.grad(loss, logits)
        ref, = torch.autograd.grad(want, z64)
        assert float((dz.double() - ref).abs().max()) <= 1e-5 * float(ref.abs().max())
    r = wb.router(logits, min(k, 32, E), mask)
    loss, counts = wb.balance_loss(logits, r.ids, mask)
    assert torch.equal(counts, r.counts) and torch.equal(loss, r.balance_loss)


def test_strided_logits_and_loss_in_place():
    logits, _ = make(90, 24)
    want = wb.router(logits, 3)
    wide = torch.full((90, 31), float("nan"), device=DEV)
    wide[:, 5:29] = logits
    for z in (wide[:, 5:29], logits.T.contiguous().T):
        r = wb.router(z, 3)
        assert torch.equal(r.weight, want.weight) and torch.equal(r.ids, want.ids) and torch.equal(r.balance_loss, want.balance_loss)
    one = wb.router(logits[:1].expand(90, 24), 3)
    assert torch.equal(one.weight, wb.router(logits[:1].repeat(90, 1), 3).weight)
    wide.requires_grad_()
    r = wb.router(wide[:, 5:29], 3)
    loss = r.balance_loss
    loss *= 0.01
    dz, = torch.autograd.grad(loss, wide)
    assert dz[:, 5:29].isfinite().all() and dz[:, 5:29].any() and not dz[:, :5].any()


def test_captured_and_replayed():
    for rows in (16, 900):
        logits, mask = make(rows, 40, padded=True)
        logits.requires_grad_()
        gw = torch.randn(rows, 4, generator=torch.Generator().manual_seed(1)).to(DEV)

        def step():
            r = wb.router(logits, 4, mask, True)
            dz, = torch.autograd.grad((r.weight * gw).sum() + r.balance_loss, logits)
            return [r.weight.detach(), r.ids, r.counts, r.balance_loss.detach(), dz]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        with torch.no_grad():
            logits.copy_(make(rows, 40, seed=5)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, step()))


def test_router_refusals():
    logits, mask = make(8, 16, padded=True)
    for args in ((logits.half(), 2), (logits[0], 1), (logits, 0), (logits, 17), (logits.cpu(), 2), (logits, 2, mask.int()), (logits, 2, mask[:7]),
                 (logits, 2, mask.cpu()), (torch.zeros(4, 257, device=DEV), 2), (torch.zeros(4, 64, device=DEV), 33)):
        with pytest.raises(ValueError):
            wb.router(*args)
    ids = torch.zeros(8, 2, dtype=torch.int32, device=DEV)
    for args in ((logits, ids.float()), (logits, ids[:7]), (logits, ids[0]), (logits, ids[:, :0]), (logits, ids.cpu()), (logits, ids, mask[:3])):
        with pytest.raises(ValueError):
            wb.balance_loss(*args)


# ---- the weighted combine --------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,k,N", [(1, 1, 1), (3, 2, 8), (130, 6, 2048), (64, 9, 1000), (500, 2, 333), (7, 5, 4104)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_combine_rows(tokens, k, N, dtype):
    g = torch.Generator().manual_seed(tokens)
    R = tokens * k + 5
    y = torch.randn(R, N, generator=g).to(dtype).to(DEV)
    row_of = torch.randperm(R, generator=g)[:tokens * k].reshape(tokens, k).to(torch.int32)
    row_of[torch.rand(tokens, k, generator=g) < 0.1] = -1
    if k > 1:
        row_of[0, 1] = row_of[0, 0]  # the same row twice
    row_of, weight, up = row_of.to(DEV), torch.randn(tokens, k, generator=g).to(DEV).requires_grad_(), torch.randn(tokens, N, generator=g).to(dtype).to(DEV)
    out = wb.combine_rows(y, row_of, weight)
    dw, = torch.autograd.grad(out, weight, up)
    rows = y.double()[row_of.long().clamp(min=0)] * (row_of >= 0)[:, :, None]
    want, size = (rows * weight.detach().double()[:, :, None]).sum(1), (rows * weight.detach().double()[:, :, None]).abs().sum(1)
    tol = size * (k + 2) * 2.0 ** -24 + want.abs() * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) + 1e-36
    assert out.dtype == dtype and bool(((out.detach().double() - want).abs() <= tol).all())
    ref, size = (rows * up.double()[:, None, :]).sum(2), (rows * up.double()[:, None, :]).abs().sum(2)
    assert bool(((dw.double() - ref).abs() <= size * (N / 128 + 32) * 2.0 ** -24 + 1e-36).all())
    assert not dw[row_of < 0].any()
    flat = torch.empty_like(out)
    moe.combine(y, row_of.reshape(-1), weight.detach().reshape(-1), k, flat)
    assert torch.equal(flat, out)
    got, = torch.autograd.grad(wb.combine_rows(y, row_of, weight).sum(), weight)  # a broadcast gradient
    assert bool(((got.double() - rows.sum(2)).abs() <= rows.abs().sum(2) * (N / 128 + 32) * 2.0 ** -24 + 1e-36).all())


def test_combine_rows_values_that_are_not_finite():
    """NaN in rows that nobody asks for, and in one that a token does."""
    y = torch.ones(6, 16, device=DEV)
    y[4:] = float("nan")
    row_of = torch.tensor([[0, 1], [2, -1], [4, 3]], dtype=torch.int32, device=DEV)
    weight = torch.ones(3, 2, device=DEV, requires_grad=True)
    out = wb.combine_rows(y, row_of, weight)
    dw, = torch.autograd.grad(out, weight, torch.ones_like(out))
    assert out[:2].isfinite().all() and out[2].isnan().all()
    assert dw[:2].tolist() == [[16.0, 16.0], [16.0, 0.0]] and dw[2, 0].isnan() and float(dw[2, 1]) == 16.0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_combine_rows_of_one_row_one_column_and_none(dtype):
    """Strides that no address depends on may be anything; without rows of y every pair is dropped."""
    one = torch.arange(1, 17, device=DEV).to(dtype)
    row_of = torch.tensor([[0, -1], [0, 0]], dtype=torch.int32, device=DEV)
    weight = torch.tensor([[2.0, 9.0], [1.0, 3.0]], device=DEV, requires_grad=True)
    for y in (one.as_strided((1, 16), (0, 1)), one.as_strided((1, 16), (5, 1))):
        out = wb.combine_rows(y, row_of, weight)
        assert torch.equal(out[0], 2 * one) and torch.equal(out[1], 4 * one)
        assert torch.autograd.grad(out.float().sum(), weight)[0].tolist() == [[136.0, 0.0], [136.0, 136.0]]
    column = one.as_strided((4, 1), (2, 7))  # 1, 3, 5, 7
    out = wb.combine_rows(column, torch.tensor([[3, 1], [0, -1]], dtype=torch.int32, device=DEV), weight)
    assert out.flatten().tolist() == [41.0, 1.0]
    assert torch.autograd.grad(out.float().sum(), weight)[0].tolist() == [[7.0, 3.0], [1.0, 0.0]]
    out = wb.combine_rows(one.reshape(1, 16)[:0], torch.full((2, 2), -1, dtype=torch.int32, device=DEV), weight)
    assert out.shape == (2, 16) and not out.any() and not torch.autograd.grad(out.float().sum(), weight)[0].any()


def test_combine_rows_refusals():
    y, row_of, weight = torch.zeros(6, 16, device=DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.zeros(3, 2, device=DEV)
    for args in ((y.half(), row_of, weight), (y, row_of.long(), weight), (y, row_of, weight.double()), (y, row_of[:2], weight), (y[0], row_of, weight),
                 (y, row_of.cpu(), weight), (y.cpu(), row_of, weight), (y, row_of[:, :0], weight[:, :0]), (y.clone().requires_grad_(), row_of, weight)):
        with pytest.raises(ValueError):
            wb.combine_rows(*args)
    assert wb.combine_rows(y, row_of[:0], weight[:0]).shape == (0, 16)


# ---- together --------------------------------------------------------------------------------------------------------------------------------


def _mlp(E, K, I, N, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    w1 = [ops.quantize_mxfp4((torch.randn(2 * I, K, generator=g) * K ** -0.5).to(DEV), want_packed=False)[:2] for _ in range(E)]
    w2 = [ops.quantize_mxfp4((torch.randn(N, I, generator=g) * I ** -0.5).to(DEV), want_packed=False)[:2] for _ in range(E)]
    return wb.MXFP4ExpertMLP([q for q, _ in w1], [s for _, s in w1], [q for q, _ in w2], [s for _, s in w2], top_k=k)


def test_expert_mlp_on_a_routing():
    """forward_routed gives what forward gives for the same choices, and the router learns through it: the gradient of a linear router behind a
    layer with adapters, from the output of the experts and the balance loss."""
    g = torch.Generator().manual_seed(1)
    T, K, E, k = 150, 256, 6, 2
    mlp = _mlp(E, K, 128, 192, k)
    x = torch.randn(T, K, generator=g).to(BF16).to(DEV)
    gate = (torch.randn(E, K, generator=g) * K ** -0.5).to(DEV).requires_grad_()
    logits = x.float() @ gate.T
    r = wb.router(logits, k)
    y = mlp.forward_routed(x, r)
    # the softmaxes differ in their last bits, so that a sum near a border may round either way: half a step each (2^-8), and 2^-20 of the terms
    steps, terms = mlp._forward_steps(x, logits.detach()).double(), 2 * mlp._expert_rows(x, r.ids)[0].double().abs().nan_to_num().max()
    assert bool(((y.detach().double() - steps).abs() <= 2 * 2.0 ** -8 * steps.abs() + 2.0 ** -20 * terms).all())
    up = torch.randn(T, 192, generator=g).to(BF16).to(DEV)
    dgate, dw = torch.autograd.grad((y.float() * up.float()).sum() + 0.1 * r.balance_loss, (gate, r.weight))
    # by hand: each expert's rows, the weights' gradient, and the router's definition in 64 bits
    rows, inverse = mlp._expert_rows(x, r.ids)
    picked = rows.double()[inverse.long().reshape(T, k)]
    ref_dw = (picked * up.double()[:, None]).sum(2)
    assert float((dw.double() - ref_dw).abs().max()) <= 1e-5 * float(ref_dw.abs().max())
    z = logits.detach().double().requires_grad_()
    weight, _, _, loss = definition(z, k, None, False, ids=r.ids)
    dz, = torch.autograd.grad((weight * ref_dw).sum() + 0.1 * loss, z)
    ref = dz.T @ x.double()
    assert float((dgate.double() - ref).norm()) <= 1e-4 * float(ref.norm())
    with pytest.raises(ValueError):
        mlp.forward_routed(x.clone().requires_grad_(), r)
    with pytest.raises(ValueError):
        mlp.forward_routed(x[:5], r)


def test_padded_rows_of_an_expert_mlp():
    g = torch.Generator().manual_seed(2)
    mlp = _mlp(4, 128, 128, 64, 2)
    x = torch.randn(40, 128, generator=g).to(BF16).to(DEV)
    logits = torch.randn(40, 4, generator=g).to(DEV)
    mask = torch.ones(40, dtype=torch.bool, device=DEV)
    mask[30:] = False
    x[30:] = float("nan")
    y = mlp.forward_routed(x, wb.router(logits, 2, mask))
    want = mlp.forward_routed(x[:30].contiguous(), wb.router(logits[:30], 2))
    assert torch.equal(y[:30], want) and not y[30:].any()


def test_block_with_adapters_router_and_experts():
    """A decode step and a training step of one block: projection with adapters, router, experts; the step's gradients reach the adapters."""
    g = torch.Generator().manual_seed(3)
    K, E = 256, 6
    proj = wb.MXFP4Linear.from_float((torch.randn(K, K, generator=g) * K ** -0.5).to(DEV))
    pool = wb.LowRankAdapters((torch.randn(3, 8, K, generator=g) * K ** -0.5).to(BF16).to(DEV), (torch.randn(3, K, 8, generator=g) * 0.1).to(BF16).to(DEV), trainable=True)
    gate = (torch.randn(E, K, generator=g) * K ** -0.5).to(DEV).requires_grad_()
    mlp = _mlp(E, K, 128, K, 2)
    for T in (1, 4, 200):
        x, ids = torch.randn(T, K, generator=g).to(BF16).to(DEV), torch.randint(-1, 3, (T,), generator=g).to(DEV)

        def block():
            h = proj(x, pool, ids)
            r = wb.router(h.float() @ gate.T, 2, renormalize=True)
            return h, r, mlp.forward_routed(h.detach(), r)

        with torch.no_grad():
            h, r, y = block()
        assert y.shape == (T, K) and y.isfinite().all() and int(r.counts.sum()) == 2 * T
        h2, r2, y2 = block()
        assert torch.equal(h2.detach(), h) and torch.equal(y2.detach(), y) and torch.equal(r2.balance_loss.detach(), r.balance_loss)
        grads = torch.autograd.grad(y2.float().square().mean() + r2.balance_loss, (gate, pool.a, pool.b))
        assert all(t.isfinite().all() for t in grads) and (T == 1 or all(t.any() for t in grads))


@pytest.mark.parametrize("tokens,k,N", [(300, 1, 1024), (70, 2, 4096), (5, 3, 1032), (40, 8, 2048), (9, 9, 2048), (20, 5, 6000)])
def test_combine_of_wide_rows_is_that_of_narrow_ones(tokens, k, N):
    """The same bits from the kernel that takes a token's whole rows and from the one that takes them in blocks of 512 columns."""
    g = torch.Generator().manual_seed(tokens)
    y, weight = torch.randn(tokens * k, N, generator=g).to(BF16).to(DEV), torch.randn(tokens, k, generator=g).to(DEV)
    row_of = torch.randperm(tokens * k, generator=g).to(torch.int32)
    row_of[::7] = -1
    row_of = row_of.to(DEV)
    wide, parts = torch.empty(tokens, N, dtype=BF16, device=DEV), torch.empty(tokens, N, dtype=BF16, device=DEV)
    moe.combine(y, row_of, weight.reshape(-1), k, wide)
    for c in range(0, N, 512):
        moe.combine(y[:, c:c + 512], row_of, weight.reshape(-1), k, parts[:, c:c + 512])
    assert torch.equal(wide, parts)
