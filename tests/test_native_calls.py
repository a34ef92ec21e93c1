"""When calls go through the host module, and when they do not because a caller watches them: runs without a GPU."""

import pytest

from wave_b200 import _lib

BESIDE = ("wb200_adapters_forward", "wb200_adapters_backward", "wb200_mxfp4_input_grad", "wb200_router", "wb200_router_grad", "wb200_moe_combine",
          "wb200_moe_combine_grad", "wb200_last_error", "wb200_router_workspace_bytes", "wb200_adapters_backward_workspace_bytes")


@pytest.fixture
def module(built_library):
    lib = _lib.load()
    assert _lib.fast(lib) is not None
    return _lib.fast(lib)


@pytest.mark.parametrize("name", BESIDE)
def test_a_function_that_is_watched_from_the_start(module, monkeypatch, name):
    """Nothing is bound while a function of the library is not the library's own, and a call of another operator does not fail for it."""
    lib = _lib.load()
    real = getattr(lib, name)
    monkeypatch.setattr(_lib, "_fast", None)
    monkeypatch.setattr(_lib, "_fast_lib", None)
    with monkeypatch.context() as m:
        m.setattr(lib, name, lambda *args: real(*args))
        assert _lib.fast() is None and _lib.native_calls() is None and _lib._fast is None
    assert _lib.native_calls() is module and _lib.unwatched(*BESIDE)  # and it is when the watching ends


@pytest.mark.parametrize("name", BESIDE)
def test_a_function_that_is_watched_later(module, monkeypatch, name):
    lib = _lib.load()
    real = getattr(lib, name)
    assert _lib.unwatched(name)
    with monkeypatch.context() as m:
        m.setattr(lib, name, lambda *args: real(*args))
        assert not _lib.unwatched(name) and not _lib.unwatched(*BESIDE)
        assert _lib.unwatched(*(other for other in BESIDE if other != name))
    assert _lib.unwatched(name)


def test_a_loader_or_a_library_that_is_replaced(module, monkeypatch):
    with monkeypatch.context() as m:
        m.setattr(_lib, "load", lambda: None)
        assert _lib.native_calls() is None
    with monkeypatch.context() as m:
        m.setattr(_lib, "_lib", object())
        assert _lib.native_calls() is None
    assert _lib.native_calls() is module
