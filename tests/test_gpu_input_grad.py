"""Input gradient of a frozen MXFP4 layer: g @ dequant(W) against the product in 64 bits.

W is exact in bf16 and so are the products in f32: what remains is the sum over N in f32 (at most (N + 8) 2^-24 of the sum of the terms' sizes, in
whatever order the tensor core adds) and the rounding to bf16 (2^-8 of the value). Tensor cores drop low bits of a term while aligning it with larger
ones: 2^-22 of the largest partial sum at each of the N / 16 steps is allowed for on top."""

import pytest
import torch

import wave_b200 as wb
from wave_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def make(M, N, K, seed=0, lo=118, hi=132):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(lo, hi, (N, K // 32), generator=g, dtype=torch.uint8)
    return torch.randn(M, N, generator=g).to(BF16).to(DEV), codes.to(DEV), scales.to(DEV)


def weight(codes, scales):
    """dequant in 64 bits, from the format's definition."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=codes.device)
    w = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).reshape(codes.shape[0], -1)
    power = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [float("nan")], dtype=torch.float64, device=codes.device)
    return w * power[scales.long()].repeat_interleave(32, 1)


def check(g, codes, scales, **kw):
    got = wb.mxfp4_input_grad(g, codes, scales, **kw)
    ops.check_device_status()
    w = weight(codes, scales)
    want, size = g.double() @ w, g.double().abs() @ w.abs()
    N = codes.shape[0]
    tol = size * ((N + 8) * 2.0 ** -24 + (N / 16 + 1) * 2.0 ** -22)
    tol = tol + (want.abs() + tol) * 2.0 ** -8 + 1e-38
    over = (got.double() - want).abs() - tol
    assert got.dtype == BF16 and bool((over <= 0).all()), f"{int((~(over <= 0)).sum())} of {over.numel()} off, by {float(over.max())}"
    return got


@pytest.mark.parametrize("M", [1, 5, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(8, 32), (64, 128), (72, 160), (200, 256), (1000, 416)])
def test_small_tiles(M, N, K):
    check(*make(M, N, K, seed=M + N))


@pytest.mark.parametrize("M,N,K", [(4096, 512, 4096), (2500, 1000, 4128), (8192, 64, 8192), (2048, 4096, 2048)])
def test_large_tiles(M, N, K):
    check(*make(M, N, K, seed=1))


@pytest.mark.parametrize("M,N,K", [(600, 4000, 2048), (16, 14336, 4096), (1, 8192, 1024), (333, 2048, 96), (128, 4096, 4096), (1024, 8192, 1024), (16, 8192, 512),
                                   (100, 8200, 2560), (250, 4096, 4064), (130, 700, 2048)])
def test_few_tiles_and_long_sums(M, N, K):
    check(*make(M, N, K, seed=2))


@pytest.mark.parametrize("N", [1, 7, 65, 1001])
def test_odd_widths(N):
    check(*make(40, N, 256, seed=3))


def test_every_code_and_scale_is_exact():
    """One nonzero per row of g picks a row of W: the result is that row rounded to bf16, which is exact for every code and scale."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)  # K = 512: every pair of codes
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    codes, scales = codes.to(DEV), scales.to(DEV)
    g = torch.eye(256, dtype=BF16, device=DEV)
    keep = torch.arange(256) < 250  # 6 * 2^127 does not fit, and 255 is NaN, which a zero of g does not stop
    got = wb.mxfp4_input_grad(g[keep][:, keep].contiguous(), codes[keep].contiguous(), scales[keep].contiguous())
    assert torch.equal(got.double(), weight(codes, scales)[keep.to(DEV)])


def test_nan_scale_spoils_its_columns_only():
    g, codes, scales = make(50, 96, 128)
    want = check(g, codes, scales)
    scales[17, 2] = 255
    got = wb.mxfp4_input_grad(g, codes, scales)
    assert got[:, 64:96].isnan().all()
    got[:, 64:96] = want[:, 64:96]
    assert torch.equal(got, want)


def test_values_that_are_not_finite_stay_in_their_rows():
    g, codes, scales = make(140, 128, 256)
    want = check(g, codes, scales)
    g[3, 5], g[130, 9] = float("nan"), float("inf")
    got = wb.mxfp4_input_grad(g, codes, scales)
    keep = torch.ones(140, dtype=torch.bool, device=DEV)
    keep[[3, 130]] = False
    assert got[3].isnan().all() and torch.equal(got[keep], want[keep]) and not got[130].isfinite().any()


def test_strides_and_given_output():
    g, codes, scales = make(70, 200, 256)
    want = check(g, codes, scales)
    wide = torch.full((70, 256), float("nan"), dtype=BF16, device=DEV)
    for at in (0, 8, 3):  # the last is copied first
        wide[:, at:at + 200] = g
        assert torch.equal(wb.mxfp4_input_grad(wide[:, at:at + 200], codes, scales), want)
        wide.fill_(float("nan"))
    assert torch.equal(wb.mxfp4_input_grad(g.T.contiguous().T, codes, scales), want)
    assert torch.equal(wb.mxfp4_input_grad(g[:1].expand(70, 200), codes, scales), wb.mxfp4_input_grad(g[:1].repeat(70, 1), codes, scales))
    pitched = torch.zeros(200, 20, dtype=torch.uint8, device=DEV)
    pitched[:, :8] = scales
    assert torch.equal(wb.mxfp4_input_grad(g, codes, pitched[:, :8]), want)
    out = torch.zeros(70, 272, dtype=BF16, device=DEV)
    assert torch.equal(wb.mxfp4_input_grad(g, codes, scales, out=out[:, 8:264]), want)
    assert torch.equal(out[:, 8:264], want) and not out[:, :8].any() and not out[:, 264:].any()
    assert wb.mxfp4_input_grad(g[:0], codes, scales).shape == (0, 256)


def test_captured_replayed_and_repeated():
    g, codes, scales = make(260, 512, 1024)
    want = check(g, codes, scales)
    assert all(torch.equal(wb.mxfp4_input_grad(g, codes, scales), want) for _ in range(20))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = wb.mxfp4_input_grad(g, codes, scales)
    new, _, _ = make(260, 512, 1024, seed=9)
    g.copy_(new)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, check(g, codes, scales))


def test_layer_gradient():
    g = torch.Generator().manual_seed(3)
    layer = wb.MXFP4Linear.from_float(torch.randn(192, 256, generator=g).to(DEV), input_grad=True)
    x = torch.randn(2, 33, 256, generator=g).to(BF16).to(DEV)
    plain = wb.MXFP4Linear(layer.weight_codes, layer.weight_scales)(x)
    x.requires_grad_()
    y = layer(x)
    up = torch.randn(2, 33, 192, generator=g).to(BF16).to(DEV)
    dx, = torch.autograd.grad(y, x, up)
    assert torch.equal(y.detach(), plain) and dx.shape == x.shape
    assert torch.equal(dx.reshape(66, 256), check(up.reshape(66, 192), layer.weight_codes, layer.weight_scales))
    got, = torch.autograd.grad(layer(x).sum(), x)  # a broadcast gradient
    assert torch.equal(got.reshape(66, 256), check(torch.ones(66, 192, dtype=BF16, device=DEV), layer.weight_codes, layer.weight_scales))
    assert not wb.MXFP4Linear(layer.weight_codes, layer.weight_scales)(x).requires_grad
    with pytest.raises(ValueError):
        layer(x.detach().float().requires_grad_())
    with pytest.raises(ValueError):
        wb.MXFP4Linear(layer.weight_codes, layer.weight_scales, torch.float32, input_grad=True)


def test_refusals():
    g, codes, scales = make(8, 64, 128)
    for args in ((g.float(), codes, scales), (g[0], codes, scales), (g[:, :63], codes, scales), (g, codes[:, :60], scales), (g, codes, scales[:, :3]),
                 (g, codes.float(), scales), (g, codes, scales.cpu()), (g, codes.cpu(), scales), (g.cpu(), codes, scales), (g, codes[0], scales)):
        with pytest.raises(ValueError):
            wb.mxfp4_input_grad(*args)
    for out in (torch.empty(8, 128, device=DEV), torch.empty(8, 127, dtype=BF16, device=DEV), torch.empty(8, 130, dtype=BF16, device=DEV)[:, 1:129],
                torch.empty(128, 8, dtype=BF16, device=DEV).T, torch.empty(8, 128, dtype=BF16)):
        with pytest.raises(ValueError):
            wb.mxfp4_input_grad(g, codes, scales, out=out)
