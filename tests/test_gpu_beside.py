"""Adapters, input gradient, router and combine as a whole: the native calls against the Python ones, threads, far offsets, parameters, derivatives
of derivatives."""

import threading

import pytest
import torch

import wave_b200 as wb
from wave_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def adapters(rows=70, K=128, N=96, rank=16, pool=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).to(DEV)  # noqa: E731
    return r(rows, N), r(rows, K), r(pool, rank, K), r(pool, N, rank), torch.randint(-1, pool, (rows,), generator=g).to(DEV), torch.rand(pool, generator=g).to(DEV)


def everything(seed=0):
    """Outputs and gradients of every operator, in order."""
    g = torch.Generator().manual_seed(seed)
    y, x, a, b, ids, s = adapters(seed=seed)
    x, a, b = (t.requires_grad_() for t in (x, a, b))
    out = wb.apply_adapters(y, x, a, b, ids, s)
    res = [out, *torch.autograd.grad(out, (x, a, b), torch.randn(70, 96, generator=g).to(BF16).to(DEV))]
    with torch.no_grad():
        res.append(wb.apply_adapters(y.float(), x, a, b, ids))
    logits = torch.randn(300, 40, generator=g).to(DEV).requires_grad_()
    mask = (torch.rand(300, generator=g) < 0.8).to(DEV)
    r = wb.router(logits, 4, mask, True)
    res += [r.weight, r.ids, r.counts, r.balance_loss, *torch.autograd.grad(r.weight.square().sum() + r.balance_loss, logits)]
    rows = torch.randn(50, 1200, generator=g).to(BF16).to(DEV)
    row_of, weight = torch.randint(-1, 50, (20, 3), generator=g, dtype=torch.int32).to(DEV), torch.rand(20, 3, generator=g).to(DEV).requires_grad_()
    out = wb.combine_rows(rows, row_of, weight)
    res += [out, *torch.autograd.grad(out, weight, torch.randn(20, 1200, generator=g).to(BF16).to(DEV))]
    codes, scales = torch.randint(0, 256, (64, 80), generator=g, dtype=torch.uint8).to(DEV), torch.randint(120, 130, (64, 5), generator=g, dtype=torch.uint8).to(DEV)
    res.append(wb.mxfp4_input_grad(torch.randn(33, 64, generator=g).to(BF16).to(DEV), codes, scales))
    return [t.detach() for t in res]


def test_native_calls_and_python_calls_agree(monkeypatch):
    assert _lib.native_calls() is not None
    native = everything()
    monkeypatch.setattr(_lib, "native_calls", lambda: None)
    assert all(torch.equal(p, q) for p, q in zip(native, everything()))


def test_native_calls_take_parameters():
    """A module's parameters are torch.nn.Parameter objects: the native call takes them too."""
    y, x, a, b, ids, s = adapters()
    pool = wb.LowRankAdapters(a, b, s, trainable=True)
    with torch.no_grad():
        assert _lib.native_calls().adapters(y, x, pool.a, pool.b, ids, pool.scale, None) is not None
    out = pool(y, x, ids)
    out.backward(torch.ones_like(out))
    want = [t.clone().requires_grad_() for t in (a, b)]
    grads = torch.autograd.grad(wb.apply_adapters(y, x, *want, ids, s), want, torch.ones_like(out))
    assert torch.equal(pool.a.grad, grads[0]) and torch.equal(pool.b.grad, grads[1])


def test_threads_with_streams_of_their_own():
    want, got = everything(), {}
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [everything() for _ in range(4)][-1]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 3 and all(torch.equal(p, q) for res in got.values() for p, q in zip(res, want))


def test_layers_and_adapters_in_two_streams_at_once():
    """Kernels that take tensor memory and wait within clusters, side by side: the same bits as one after the other."""
    g = torch.Generator().manual_seed(2)
    layer = wb.MXFP4Linear.from_float((torch.randn(4096, 4096, generator=g) / 64).to(DEV), input_grad=True)
    xs = [torch.randn(rows, 4096, generator=g).to(BF16).to(DEV) for rows in (8, 500, 4096)]
    a, b = (torch.randn(6, 64, 4096, generator=g) / 64).to(BF16).to(DEV), (torch.randn(6, 4096, 64, generator=g) / 8).to(BF16).to(DEV)
    ids = [torch.randint(-1, 6, (x.shape[0],), generator=g).sort().values.to(DEV) for x in xs]
    works = [lambda: [layer(x) for x in xs] + [wb.mxfp4_input_grad(x, layer.weight_codes, layer.weight_scales) for x in xs],
             lambda: [wb.apply_adapters(x, x, a, b, i) for x, i in zip(xs, ids)]]
    want = [work() for work in works]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for stream, work in zip(streams, works):
            with torch.cuda.stream(stream):
                got.append(work())
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for one, other in zip(got, want) for p, q in zip(one, other))
    wb.ops.check_device_status()


@pytest.mark.parametrize("python", [False, True])
def test_a_derivative_of_a_derivative_is_refused(python, monkeypatch):
    if python:
        monkeypatch.setattr(_lib, "native_calls", lambda: None)
    y, x, a, b, ids, s = adapters()
    x, a, b = (t.requires_grad_() for t in (x, a, b))
    grads = torch.autograd.grad(wb.apply_adapters(y, x, a, b, ids, s).float().square().sum(), (x, a, b), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grads[0].float().sum(), a)
    logits = torch.randn(9, 8, device=DEV, requires_grad=True)
    dz, = torch.autograd.grad(wb.router(logits, 2).balance_loss, logits, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dz.sum(), logits)


def test_a_tensor_changed_before_the_backward_pass_is_noticed():
    y, x, a, b, ids, s = adapters()
    x, a = x.requires_grad_(), a.requires_grad_()
    out = wb.apply_adapters(y, x, a, b, ids, s)
    ids.fill_(0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.float().sum(), (x, a))


def test_rows_behind_32_bit_offsets():
    """y and out of 2.4e9 elements; x of as few as may be."""
    rows, K, N = 75_000, 8, 32_768
    g = torch.Generator().manual_seed(1)
    x, a, b = torch.randn(rows, K, generator=g).to(BF16).to(DEV), torch.randn(2, 16, K, generator=g).to(BF16).to(DEV), torch.randn(2, N, 16, generator=g).to(BF16).to(DEV)
    ids = (torch.arange(rows) % 3 - 1).to(DEV)
    y = torch.zeros(rows, N, dtype=BF16, device=DEV)
    y[-100:] = 1.0
    out = wb.apply_adapters(y, x, a, b, ids)
    for part in (slice(0, 100), slice(65_500, 65_600), slice(-100, None)):
        assert torch.equal(out[part], wb.apply_adapters(y[part].contiguous(), x[part].contiguous(), a, b, ids[part].contiguous()))
    del y, out
    torch.cuda.empty_cache()


def test_adapters_behind_32_bit_offsets():
    pool, rank, K, N = 36_000, 8, 8_192, 64
    a, b = torch.zeros(pool, rank, K, dtype=BF16, device=DEV), torch.zeros(pool, N, rank, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(2)
    a[-3:], b[-3:] = torch.randn(3, rank, K, generator=g).to(BF16).to(DEV), torch.randn(3, N, rank, generator=g).to(BF16).to(DEV)
    for rows in (9, 100):
        x, y = torch.randn(rows, K, generator=g).to(BF16).to(DEV), torch.randn(rows, N, generator=g).to(BF16).to(DEV)
        ids = torch.randint(pool - 3, pool, (rows,), generator=g).to(DEV)
        near = wb.apply_adapters(y, x, a[-3:].contiguous(), b[-3:].contiguous(), ids - (pool - 3))
        assert torch.equal(wb.apply_adapters(y, x, a, b, ids), near)
    del a, b
    torch.cuda.empty_cache()


def test_a_training_step_through_backward_and_in_a_graph():
    """.backward() into parameters, then the same step captured (no graph of the eager step alive) and replayed."""
    y, x, a, b, ids, s = adapters(rows=200)
    pool = wb.LowRankAdapters(a, b, s, trainable=True)
    g = torch.randn(200, 96, generator=torch.Generator().manual_seed(3)).to(BF16).to(DEV)

    def step():
        pool.zero_grad(set_to_none=True)
        pool(y, x, ids).backward(g)
        return pool.a.grad, pool.b.grad

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    pool.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
