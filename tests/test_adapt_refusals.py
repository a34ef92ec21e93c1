"""What the C entry points of adapters, input gradient, router and combine refuse before they touch a device: runs without a GPU."""

import pytest

from wave_b200 import _lib

P = 0x10000  # an address that nothing reads: every call here is refused


@pytest.fixture(scope="module")
def lib(built_library):
    return _lib.load()


def refused(lib, rc, code, words):
    message = lib.wb200_last_error().decode()
    assert rc == code and words in message, (rc, message)


def adapters_args(**kw):
    a = dict(rows=4, K=64, N=32, rank=8, pool=2, x=P, ldx=64, a=P, b=P, ids=P, wide=0, scale=None, y=P, ldy=32, out=P, ldo=32, dtype=_lib.WB200_BF16, hidden=P,
             nbytes=1 << 20, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(rows=0), _lib.WB200_ERR_INVALID_ARG, "rows = 0"), (dict(K=60), _lib.WB200_ERR_INVALID_ARG, "multiple of 8"),
    (dict(rank=257), _lib.WB200_ERR_UNSUPPORTED, "above 256"), (dict(rows=5000000), _lib.WB200_ERR_UNSUPPORTED, "rows in one call"),
    (dict(N=9000000), _lib.WB200_ERR_UNSUPPORTED, "too wide"), (dict(x=None), _lib.WB200_ERR_INVALID_ARG, "null pointer"),
    (dict(hidden=None), _lib.WB200_ERR_INVALID_ARG, "null pointer"), (dict(dtype=7), _lib.WB200_ERR_INVALID_ARG, "unknown output dtype"),
    (dict(ldy=31), _lib.WB200_ERR_INVALID_ARG, "pitch is smaller"), (dict(ldy=1 << 24), _lib.WB200_ERR_UNSUPPORTED, "2^24"),
    (dict(y=P + 1), _lib.WB200_ERR_ALIGNMENT, "aligned"), (dict(ids=P + 4, wide=1), _lib.WB200_ERR_ALIGNMENT, "aligned"),
    (dict(nbytes=4 * 2 * 16 * 2 - 1), _lib.WB200_ERR_WORKSPACE, "hidden of 256 bytes"),
])
def test_adapters_forward(lib, kw, code, words):
    refused(lib, lib.wb200_adapters_forward(*adapters_args(**kw)), code, words)


def backward_args(**kw):
    a = dict(rows=4, K=64, N=33, rank=8, pool=2, x=P, ldx=64, a=P, b=P, ids=P, wide=0, scale=None, g=P, ldg=33, hidden=P, hidden_bytes=1 << 20, dx=P, ldd=64,
             accumulate=0, da=P, db=P, ws=P, ws_bytes=1 << 20, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(pool=65536), _lib.WB200_ERR_UNSUPPORTED, "65535"), (dict(dx=None, da=None, db=None), _lib.WB200_ERR_INVALID_ARG, "no gradient"),
    (dict(g=None), _lib.WB200_ERR_INVALID_ARG, "null pointer"), (dict(ws=None), _lib.WB200_ERR_INVALID_ARG, "null pointer"),
    (dict(hidden=None), _lib.WB200_ERR_INVALID_ARG, "null pointer"), (dict(ldg=32), _lib.WB200_ERR_INVALID_ARG, "pitch is smaller"),
    (dict(ldd=1 << 24), _lib.WB200_ERR_UNSUPPORTED, "2^24"), (dict(ws=P + 8), _lib.WB200_ERR_ALIGNMENT, "aligned"),
    (dict(ws_bytes=255), _lib.WB200_ERR_WORKSPACE, "workspace of 576 bytes"), (dict(hidden_bytes=255), _lib.WB200_ERR_WORKSPACE, "hidden of 256 bytes"),
])
def test_adapters_backward(lib, kw, code, words):
    refused(lib, lib.wb200_adapters_backward(*backward_args(**kw)), code, words)


def test_sizes(lib):
    assert lib.wb200_adapters_hidden_bytes(5, 17, _lib.WB200_BF16) == 5 * 2 * 32 * 2 and lib.wb200_adapters_hidden_bytes(5, 17, _lib.WB200_F32) == 5 * 3 * 32 * 2
    assert lib.wb200_adapters_hidden_bytes(0, 17, 0) == 0 and lib.wb200_adapters_hidden_bytes(5, 0, 0) == 0
    assert lib.wb200_adapters_backward_workspace_bytes(4, 32, 8) == 256 and lib.wb200_adapters_backward_workspace_bytes(4, 33, 8) == 256 + 4 * 40 * 2
    assert lib.wb200_router_workspace_bytes(64, 8) == 4 * 17 and lib.wb200_router_workspace_bytes(0, 8) == 0


def grad_args(**kw):
    a = dict(M=4, N=64, K=64, g=P, ldg=64, b=P, s=P, lds=2, dx=P, ldd=64, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(M=0), _lib.WB200_ERR_INVALID_ARG, "positive"), (dict(K=48), _lib.WB200_ERR_INVALID_ARG, "group size"), (dict(dx=None), _lib.WB200_ERR_INVALID_ARG, "null"),
    (dict(ldg=56), _lib.WB200_ERR_INVALID_ARG, "pitch"), (dict(lds=1), _lib.WB200_ERR_INVALID_ARG, "pitch"), (dict(ldg=65), _lib.WB200_ERR_ALIGNMENT, "aligned"),
    (dict(g=P + 8), _lib.WB200_ERR_ALIGNMENT, "aligned"), (dict(b=P + 8), _lib.WB200_ERR_ALIGNMENT, "aligned"), (dict(ldd=68), _lib.WB200_ERR_ALIGNMENT, "aligned"),
])
def test_input_grad(lib, kw, code, words):
    refused(lib, lib.wb200_mxfp4_input_grad(*grad_args(**kw)), code, words)


def router_args(**kw):
    a = dict(rows=4, E=8, k=2, logits=P, dtype=_lib.WB200_F32, ld=8, mask=None, given=None, wide=0, renorm=0, weight=P, ids=P, counts=P, unit=P, loss=P, ws=P,
             nbytes=1 << 20, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(rows=0), _lib.WB200_ERR_INVALID_ARG, "rows = 0"), (dict(E=257, ld=257), _lib.WB200_ERR_UNSUPPORTED, "at most 256"),
    (dict(k=9), _lib.WB200_ERR_INVALID_ARG, "top_k = 9"), (dict(E=64, ld=64, k=33), _lib.WB200_ERR_INVALID_ARG, "top_k = 33"),
    (dict(dtype=9), _lib.WB200_ERR_INVALID_ARG, "dtype"), (dict(ld=7), _lib.WB200_ERR_INVALID_ARG, "pitch"), (dict(logits=P + 2), _lib.WB200_ERR_ALIGNMENT, "aligned"),
    (dict(weight=None), _lib.WB200_ERR_INVALID_ARG, "null"), (dict(loss=None), _lib.WB200_ERR_INVALID_ARG, "null"), (dict(nbytes=67), _lib.WB200_ERR_WORKSPACE, "68 bytes"),
    (dict(rows=(1 << 30) + 1, k=1), _lib.WB200_ERR_UNSUPPORTED, "in one call"), (dict(rows=1 << 30, k=2), _lib.WB200_ERR_UNSUPPORTED, "in one call"),
])
def test_router(lib, kw, code, words):
    refused(lib, lib.wb200_router(*router_args(**kw)), code, words)


def test_router_grad_and_combine_grad(lib):
    ok = [4, 8, 2, P, _lib.WB200_F32, 8, None, P, P, P, 0, P, P, P, 8, None]
    for at, value, words in ((7, None, "null"), (11, None, "null"), (12, None, "null"), (13, None, "null"), (14, 7, "pitch"), (2, 9, "top_k")):
        refused(lib, lib.wb200_router_grad(*[value if i == at else v for i, v in enumerate(ok)]), _lib.WB200_ERR_INVALID_ARG, words)
    ok = [P, 32, P, 32, _lib.WB200_BF16, P, 4, 2, 32, P, None]
    for at, value, words in ((0, None, "null"), (1, 31, "pitch"), (3, 31, "pitch"), (4, 5, "dtype"), (6, 0, "tokens = 0"), (9, None, "null")):
        refused(lib, lib.wb200_moe_combine_grad(*[value if i == at else v for i, v in enumerate(ok)]), _lib.WB200_ERR_INVALID_ARG, words)


def test_front_ends_refuse_cpu_tensors(lib):
    import torch

    import wave_b200 as wb
    z = torch.zeros
    b = torch.bfloat16
    for call in (lambda: wb.apply_adapters(z(2, 8, dtype=b), z(2, 8, dtype=b), z(1, 4, 8, dtype=b), z(1, 8, 4, dtype=b), z(2, dtype=torch.int32)),
                 lambda: wb.mxfp4_input_grad(z(2, 8, dtype=b), z(8, 16, dtype=torch.uint8), z(8, 1, dtype=torch.uint8)), lambda: wb.router(z(2, 4), 1),
                 lambda: wb.balance_loss(z(2, 4), z(2, 1, dtype=torch.int32)), lambda: wb.combine_rows(z(2, 4), z(1, 1, dtype=torch.int32), z(1, 1))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        wb.LowRankAdapters(z(2, 4, 8, dtype=b), z(2, 8, 3, dtype=b))
