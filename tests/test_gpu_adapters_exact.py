"""The adapters' hidden vectors A x and B^T g are f32 sums, and nothing of them is lost before the second product: shown on values for which every
product and every sum, in any order, is exact in f32, so that the results are known to the last bit.

The hidden numbers are 1 + 2^-9 + 2^-20 and 1 + 2^-9 (21 and 10 bits of a significand of 24). Their difference, 2^-20, is a bf16 number; it is lost as soon
as one of them is held in fewer than 21 bits."""

import pytest
import torch

import wave_b200 as wb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
LONG, SHORT = (1.0, 2.0 ** -9, 2.0 ** -20), (1.0, 2.0 ** -9)

# rows, K, N, rank, pool: few rows (whole ranks, others), chunks of 64 rows (aligned or not, every number of rank steps), the tensor cores
SIZES = [(1, 64, 64, 16, 4), (3, 256, 200, 8, 5), (5, 64, 40, 32, 3), (7, 128, 72, 64, 9), (4, 64, 33, 12, 2), (20, 4096, 24, 20, 40),
         (200, 256, 264, 16, 2), (130, 520, 96, 32, 3), (300, 64, 200, 64, 1), (90, 128, 100, 7, 2), (75, 64, 33, 40, 2), (200, 256, 128, 100, 3), (150, 96, 64, 256, 1),
         (2100, 512, 136, 16, 3), (2100, 512, 40, 24, 3), (300, 1024, 72, 48, 2), (8200, 64, 4104, 64, 3), (8400, 4160, 64, 48, 2)]


def pool_of(rows, rank, pool):
    """Ids in runs, every adapter among them where there are rows enough; the two ranks that hold something."""
    ids = (torch.arange(rows, device=DEV) * min(pool, rows) // rows).to(torch.int32)
    return ids, 0, rank - 1


def wide(length, values):
    v = torch.zeros(length, dtype=BF16, device=DEV)
    v[:len(values)] = torch.tensor(values, dtype=BF16)
    return v


@pytest.mark.parametrize("rows,K,N,rank,pool", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_output(rows, K, N, rank, pool, dtype):
    ids, p, q = pool_of(rows, rank, pool)
    a, b = torch.zeros(pool, rank, K, dtype=BF16, device=DEV), torch.zeros(pool, N, rank, dtype=BF16, device=DEV)
    a[:, p], a[:, q] = wide(K, LONG), wide(K, SHORT)
    b[:, :, p], b[:, :, q] = 1, -1
    x = torch.ones(rows, K, dtype=BF16, device=DEV)
    got = wb.apply_adapters(torch.zeros(rows, N, dtype=dtype, device=DEV), x, a, b, ids)
    assert torch.equal(got, torch.full_like(got, 2.0 ** -20))


@pytest.mark.parametrize("rows,K,N,rank,pool", SIZES)
def test_input_gradient(rows, K, N, rank, pool):
    ids, p, q = pool_of(rows, rank, pool)
    a, b = torch.zeros(pool, rank, K, dtype=BF16, device=DEV), torch.zeros(pool, N, rank, dtype=BF16, device=DEV)
    b[:, :, p], b[:, :, q] = wide(N, LONG), wide(N, SHORT)
    a[:, p], a[:, q] = 1, -1
    x = torch.zeros(rows, K, dtype=BF16, device=DEV, requires_grad=True)
    out = wb.apply_adapters(torch.zeros(rows, N, dtype=BF16, device=DEV), x, a, b, ids)
    dx, = torch.autograd.grad(out, x, torch.ones_like(out))
    assert torch.equal(dx, torch.full_like(dx, 2.0 ** -20))


@pytest.mark.parametrize("rows,K,N,rank,pool", [s for s in SIZES if s[0] > 1])
def test_gradients_of_the_adapter(rows, K, N, rank, pool):
    """The first and the last row of one adapter, with opposite signs; the rows between them add nothing."""
    ids, p, _ = pool_of(rows, rank, pool)
    ids[0] = ids[-1] = 1 % pool
    sides = torch.zeros(rows, 1, dtype=BF16, device=DEV)
    sides[0], sides[-1] = 1, -1

    def ends(length):
        t = torch.zeros(rows, length, dtype=BF16, device=DEV)
        t[0, :3] = t[-1, :2] = 1
        return t

    # of a: u = B^T g is LONG and SHORT in the two rows, x is 1 and -1
    a, b = torch.zeros(pool, rank, K, dtype=BF16, device=DEV, requires_grad=True), torch.zeros(pool, N, rank, dtype=BF16, device=DEV)
    b[:, :, p] = wide(N, LONG)
    out = wb.apply_adapters(torch.zeros(rows, N, dtype=BF16, device=DEV), sides.expand(rows, K).contiguous(), a, b, ids)
    da, = torch.autograd.grad(out, a, ends(N))
    want = torch.zeros_like(da)
    want[1 % pool, p] = 2.0 ** -20
    assert torch.equal(da, want)
    # of b: A x is LONG and SHORT, g is 1 and -1
    a, b = torch.zeros(pool, rank, K, dtype=BF16, device=DEV), torch.zeros(pool, N, rank, dtype=BF16, device=DEV, requires_grad=True)
    a[:, p] = wide(K, LONG)
    out = wb.apply_adapters(torch.zeros(rows, N, dtype=BF16, device=DEV), ends(K), a, b, ids)
    db, = torch.autograd.grad(out, b, sides.expand(rows, N).contiguous())
    want = torch.zeros_like(db)
    want[1 % pool, :, p] = 2.0 ** -20
    assert torch.equal(db, want)
