"""Edges of the calls beside frozen weights: what is dropped, watched, written in place or differentiated in another way."""

import ctypes
import sys
import threading

import pytest
import torch

import wave_b200 as wb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_combine_without_rows_drops_pairs_of_any_weight(dtype, value):
    """Without rows of y every pair is dropped, and a dropped pair adds nothing whatever its weight: as with rows and all pairs -1."""
    row_of = torch.full((3, 2), -1, dtype=torch.int32, device=DEV)
    weight = torch.rand(3, 2, device=DEV)
    weight[1, 0] = value
    weight.requires_grad_()
    for rows in (0, 4):
        out = wb.combine_rows(torch.ones(rows, 16, dtype=dtype, device=DEV), row_of, weight)
        assert out.dtype == dtype and torch.equal(out, torch.zeros_like(out))
        grad, = torch.autograd.grad(out, weight, torch.ones_like(out))
        assert torch.equal(grad, torch.zeros_like(grad))


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor's tangent would be dropped in silence: every call refuses it, in native code and without."""
    import torch.autograd.forward_ad as fwd

    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    y, x, a, b = r(4, 32).to(BF16), r(4, 64).to(BF16), r(2, 8, 64).to(BF16), r(2, 32, 8).to(BF16)
    ids, logits = torch.zeros(4, dtype=torch.int32, device=DEV), r(4, 8)
    row_of, weight = torch.zeros(4, 2, dtype=torch.int32, device=DEV), r(4, 2)
    layer = wb.MXFP4Linear.from_float(r(32, 64), input_grad=True)
    pool = wb.LowRankAdapters(a, b)
    codes, scales = layer.weight_codes, layer.weight_scales
    experts = wb.MXFP4ExpertMLP(*[list(torch.zeros(s, dtype=torch.uint8, device=DEV)) for s in ((2, 256, 32), (2, 256, 2), (2, 64, 64), (2, 64, 4))], top_k=2)
    routing = wb.Routing(weight, row_of, ids, logits.sum())
    calls = [(y, lambda d: wb.apply_adapters(d, x, a, b, ids)), (x, lambda d: wb.apply_adapters(y, d, a, b, ids)), (a, lambda d: wb.apply_adapters(y, x, d, b, ids)),
             (b, lambda d: wb.apply_adapters(y, x, a, d, ids)), (logits, lambda d: wb.router(d, 2)), (logits, lambda d: wb.balance_loss(d, row_of)),
             (y, lambda d: wb.combine_rows(d, row_of, weight)), (weight, lambda d: wb.combine_rows(y, row_of, d)), (y, lambda d: wb.mxfp4_input_grad(d, codes, scales)),
             (x, lambda d: layer(d)), (x, lambda d: layer(d, pool, ids)), (x, lambda d: experts.forward_routed(d, routing))]
    for native in (True, False):
        if not native:
            monkeypatch.setattr(wb._lib, "native_calls", lambda: None)
        for tensor, call in calls:
            call(tensor)
            with fwd.dual_level():
                with pytest.raises(ValueError, match="forward-mode"):
                    call(fwd.make_dual(tensor, torch.ones_like(tensor)))
                call(tensor)  # one without a tangent, at the same time


@pytest.mark.parametrize("native", [True, False])
def test_a_given_output_counts_as_changed(native, monkeypatch):
    """An operator that kept y for its backward pass learns that y was written over, as by an in-place operation of torch; an out that is part of a graph
    is refused."""
    if not native:
        monkeypatch.setattr(wb._lib, "native_calls", lambda: None)
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).to(DEV)  # noqa: E731
    y, x, a, b, ids = r(6, 32), r(6, 64), r(2, 8, 64), r(2, 32, 8), torch.zeros(6, dtype=torch.int32, device=DEV)
    w = r(6, 32).requires_grad_()
    layer = wb.MXFP4Linear.from_float(torch.randn(32, 64, generator=g).to(DEV))
    up = y.clone()
    for kept, change in ((y, lambda t: wb.apply_adapters(t, x, a, b, ids, out=t)), (y, lambda t: wb.apply_adapters(y.clone(), x, a, b, ids, out=t)),
                         (r(6, 64), lambda t: wb.mxfp4_input_grad(up, layer.weight_codes, layer.weight_scales, out=t))):
        z = kept * (w if kept.shape == w.shape else w[:, :1])
        with torch.no_grad():
            change(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        assert w.grad is None
        z = kept * (w if kept.shape == w.shape else w[:, :1])
        z.sum().backward()
        w.grad = None
        leaf = kept.clone().requires_grad_()
        with pytest.raises(ValueError):
            change(leaf)
        with torch.inference_mode():  # a tensor without a version
            change(kept.clone())


def test_a_call_that_makes_its_output_changes_none():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).to(DEV)  # noqa: E731
    args = r(6, 32), r(6, 64), r(2, 8, 64), r(2, 32, 8), torch.zeros(6, dtype=torch.int32, device=DEV)
    before = [t._version for t in args]
    out = wb.apply_adapters(*args)
    assert [t._version for t in args] == before and out._version == 0


def test_watched_functions_of_the_library_are_called(monkeypatch):
    """A wrapper around one of the library's functions sees the calls and the backward passes of an operator, from the next call on."""
    lib, seen = wb._lib.load(), []

    def watch(name):
        real = getattr(lib, name)
        monkeypatch.setattr(lib, name, lambda *args: (seen.append(name), real(*args))[1])

    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    y, x, a, b, ids = r(4, 32).to(BF16), r(4, 64).to(BF16), r(2, 8, 64).to(BF16).requires_grad_(), r(2, 32, 8).to(BF16), torch.zeros(4, dtype=torch.int32, device=DEV)
    logits, weight = r(4, 8).requires_grad_(), r(4, 2).requires_grad_()
    layer = wb.MXFP4Linear.from_float(r(32, 64))
    calls = {"wb200_adapters_forward": lambda: wb.apply_adapters(y, x, a, b, ids), "wb200_router": lambda: wb.router(logits, 2).weight,
             "wb200_moe_combine": lambda: wb.combine_rows(y, torch.zeros(4, 2, dtype=torch.int32, device=DEV), weight),
             "wb200_mxfp4_input_grad": lambda: wb.mxfp4_input_grad(y, layer.weight_codes, layer.weight_scales)}
    backward = {"wb200_adapters_forward": "wb200_adapters_backward", "wb200_router": "wb200_router_grad", "wb200_moe_combine": "wb200_moe_combine_grad"}
    want = {name: call().detach() for name, call in calls.items()}
    for name in [*calls, *backward.values()]:
        watch(name)
    for name, call in calls.items():
        seen.clear()
        out = call()
        assert seen == [name] and torch.equal(out, want[name])
        if name in backward:
            out.sum().backward()
            assert seen == [name, backward[name]]


def test_the_interpreter_lock_is_given_back_around_launches():
    """In the place of every entry that launches, the host module gets Python's own question whether this thread holds the lock: a yes is an error status."""
    lib, module = wb._lib.load(), wb._lib.fast()
    names = ("wb200_adapters_forward", "wb200_adapters_backward", "wb200_mxfp4_input_grad", "wb200_router_workspace_bytes", "wb200_router", "wb200_router_grad",
             "wb200_moe_combine", "wb200_moe_combine_grad", "wb200_last_error", "wb200_adapters_backward_workspace_bytes")
    asked = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
    own = [ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in names]
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    y, x, a, b, ids = r(4, 32).to(BF16), r(4, 64).to(BF16), r(2, 8, 64).to(BF16), r(2, 32, 8).to(BF16), torch.zeros(4, dtype=torch.int32, device=DEV)
    row_of = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    layer = wb.MXFP4Linear.from_float(r(32, 64))
    module.bind_adapt(*(p if name.endswith(("_bytes", "_error")) else asked for name, p in zip(names, own)))
    try:
        wb.mxfp4_input_grad(y, layer.weight_codes, layer.weight_scales)
        for trained in (False, True):
            leaf, logits, weight = a.clone().requires_grad_(trained), r(4, 8).requires_grad_(trained), r(4, 2).requires_grad_(trained)
            outs = wb.apply_adapters(y, x, leaf, b, ids), wb.router(logits, 2).weight, wb.combine_rows(y, row_of, weight)
            if trained:
                for out in outs:
                    out.sum().backward()
        wb.apply_adapters(y, x, a, b, ids, out=y)
    finally:
        module.bind_adapt(*own)
    assert ctypes.pythonapi.PyGILState_Check() == 1  # and it is held again


def test_a_layer_without_adapters_is_called_as_directly_as_before():
    """Of the package's Python functions only forward itself and the question for the host module run in front of the native call."""
    layer = wb.MXFP4Linear.from_float(torch.randn(64, 128, device=DEV))
    x = torch.randn(4, 128, device=DEV).to(BF16)
    want = layer(x)
    seen = []
    sys.setprofile(lambda frame, event, arg: seen.append(frame.f_code.co_name) if event == "call" and "wave_b200" in frame.f_code.co_filename else None)
    try:
        got = layer(x)
    finally:
        sys.setprofile(None)
    assert seen == ["forward", "_native"] and torch.equal(got, want)


@pytest.mark.parametrize("tokens,cols,by_token", [(1, 4096, True), (1, 8192, False), (255, 8192, False), (256, 8192, True), (3, 16384, False), (512, 16384, True), (4, 512, False)])
@pytest.mark.parametrize("top_k", [1, 6, 8])
def test_few_tokens_of_wide_rows_are_combined_by_all_threads_at_once(tokens, cols, by_token, top_k):
    """Which of its two kernels the sum of a token's rows takes, and that the result is the same on both sides of the border: f32 sums in slot order, at most
    one rounding for each of top_k products and sums, and one to bf16."""
    g = torch.Generator().manual_seed(tokens)
    y = torch.randn(tokens * top_k + 3, cols, generator=g).to(BF16).to(DEV)
    row_of = torch.randperm(tokens * top_k + 3, generator=g)[:tokens * top_k].reshape(tokens, top_k).to(torch.int32).to(DEV)
    row_of[0, top_k // 2] = -1
    weight = torch.rand(tokens, top_k, generator=g).to(DEV)
    wb.combine_rows(y, row_of, weight)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        got = wb.combine_rows(y, row_of, weight)
        torch.cuda.synchronize()
    names = " ".join(e.key for e in prof.key_averages())
    assert ("combine_token_kernel" in names) == by_token and ("moe_combine_kernel" in names) != by_token, names
    rows = y.double()[row_of.clamp(min=0).long()] * (row_of >= 0).double()[:, :, None] * weight.double()[:, :, None]
    want, size = rows.sum(1), rows.abs().sum(1)
    tol = 2 * top_k * 2.0 ** -24 * size
    tol = tol + 2.0 ** -8 * (want.abs() + tol) + 1e-38
    assert bool(((got.double() - want).abs() <= tol).all())


def training_call(seed):
    """A call of every operator with its gradients, on inputs made from the seed: () -> the outputs and gradients."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    y, x, a, b = (t.to(BF16).requires_grad_() for t in (r(90, 40), r(90, 64), r(3, 8, 64), r(3, 40, 8)))
    ids = torch.randint(-1, 3, (90,), generator=g).to(torch.int32).to(DEV)
    logits, weight = r(90, 12).requires_grad_(), r(30, 3).requires_grad_()
    row_of, rows = torch.randperm(90, generator=g).to(torch.int32).to(DEV).reshape(30, 3), r(90, 40).to(BF16)

    def call():
        routing = wb.router(logits, 2)
        outs = [wb.apply_adapters(y, x, a, b, ids), routing.weight, routing.balance_loss, wb.combine_rows(rows, row_of, weight)]
        grads = torch.autograd.grad(outs, (y, x, a, b, logits, weight), [torch.ones_like(o) for o in outs])
        return [o.detach() for o in outs] + list(grads)

    return call


def test_saved_tensors_pass_through_hooks():
    """Python functions that pack and unpack what is saved run while a native call builds its node."""
    call = training_call(3)
    want = call()
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(p, q) for p, q in zip(call(), want))
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(tuple(t.shape)), t.clone())[1], lambda t: t):
        assert all(torch.equal(p, q) for p, q in zip(call(), want))
    assert (90, 64) in seen and (90, 12) in seen and (90, 40) in seen
    with torch.autograd.set_detect_anomaly(True):
        assert all(torch.equal(p, q) for p, q in zip(call(), want))


def test_threads_call_at_once():
    """Calls with gradients from several threads, each on a stream and on inputs of its own."""
    calls = [training_call(seed) for seed in range(4)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(25):
                    got = calls[i]()
                stream.synchronize()
            if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not bad and not any(t.is_alive() for t in threads)
