"""Every pointer that the C entries beside frozen weights take has to be aligned to its elements: refused before a device is touched, runs without a GPU."""

import pytest

from wave_b200 import _lib

P = 0x10000  # an address that nothing reads: every call here is refused


@pytest.fixture(scope="module")
def lib(built_library):
    return _lib.load()


def refused(lib, call, args, at, off):
    rc = getattr(lib, call)(*[v + off if i == at else v for i, v in enumerate(args)])
    assert rc == _lib.WB200_ERR_ALIGNMENT and "aligned" in lib.wb200_last_error().decode(), (call, at, off, rc)


FORWARD = [4, 64, 32, 8, 2, P, 64, P, P, P, 0, P, P, 32, P, 32, _lib.WB200_F32, P, 1 << 20, None]
BACKWARD = [4, 64, 33, 8, 2, P, 64, P, P, P, 0, P, P, 33, P, 1 << 20, P, 64, 0, P, P, P, 1 << 20, None]
ROUTER = [4, 8, 2, P, _lib.WB200_F32, 8, None, None, 0, 0, P, P, P, P, P, P, 1 << 20, None]
GIVEN = [4, 8, 2, P, _lib.WB200_BF16, 8, None, P, 1, 0, None, None, P, P, P, P, 1 << 20, None]
ROUTER_GRAD = [4, 8, 2, P, _lib.WB200_F32, 8, None, P, P, P, 0, P, P, P, 8, None]
COMBINE_GRAD = [P, 32, P, 32, _lib.WB200_F32, P, 4, 2, 32, P, None]


@pytest.mark.parametrize("call,args,at,off", [
    *(("wb200_adapters_forward", FORWARD, at, off) for at, off in ((5, 1), (7, 1), (8, 1), (9, 2), (11, 2), (12, 2), (14, 2), (17, 8))),
    *(("wb200_adapters_backward", BACKWARD, at, off) for at, off in ((5, 1), (7, 1), (8, 1), (9, 2), (11, 2), (12, 1), (14, 8), (16, 1), (19, 1), (20, 1), (21, 8))),
    *(("wb200_router", ROUTER, at, 2) for at in (3, 10, 11, 12, 13, 14, 15)),
    *(("wb200_router", GIVEN, at, off) for at, off in ((3, 1), (7, 4), (12, 2), (14, 1))),
    *(("wb200_router_grad", ROUTER_GRAD, at, 2) for at in (3, 7, 8, 9, 11, 12, 13)),
    *(("wb200_moe_combine_grad", COMBINE_GRAD, at, 2) for at in (0, 2, 5, 9)),
])
def test_pointers_between_elements_are_refused(lib, call, args, at, off):
    refused(lib, call, args, at, off)
