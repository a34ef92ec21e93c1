"""Edges of the calls beside frozen weights: what is dropped, watched, written in place or differentiated in another way."""

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
