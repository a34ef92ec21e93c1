"""Low-rank adapters of many requests beside a shared projection.

    out[t] = y[t] + scale[l] * B_l (A_l x[t]),   l = ids[t]

Every row picks its own adapter from a pool, or none; rows need no order. The reference has no adapters; its module wrappers
(wave_lang/kernel/wave/nn/linear.py:147) are where they would sit, as they sit on `MXFP4Linear` here. Forward for serving and
training, with the gradients of x, a and b through autograd; the kernels are csrc/adapters.cuh.
"""

from __future__ import annotations

import torch

from . import _lib, ops

_OUT_CODE = ops._DTYPE_CODE
MAX_RANK = 256
MAX_TRAINED = 65535  # adapters of a pool whose gradients are asked for


def _check(y, x, a, b, ids, scale, out) -> tuple[int, int, int, int, int]:
    """(rows, K, N, rank, adapters); everything that would make the kernels read or write elsewhere is refused."""
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor; wave_b200 has no CPU path")
    ops.refuse_tangents(y, x, a, b, scale)
    if x.dtype != torch.bfloat16 or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise ValueError(f"x, a and b must be bfloat16, got {x.dtype}, {a.dtype} and {b.dtype}")
    if x.dim() != 2 or y.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError("x and y must be 2-D, a [adapters, rank, K] and b [adapters, N, rank]")
    rows, K = x.shape
    pool, rank, _ = a.shape
    N = y.shape[1]
    if y.shape[0] != rows or a.shape[2] != K or tuple(b.shape) != (pool, N, rank):
        raise ValueError(f"shapes do not agree: y {tuple(y.shape)}, x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)}")
    if y.dtype not in _OUT_CODE:
        raise ValueError(f"y must be float32 or bfloat16, got {y.dtype}")
    if ids.dtype not in (torch.int32, torch.int64) or tuple(ids.shape) != (rows,):
        raise ValueError(f"ids must be int32 or int64 [{rows}], got {ids.dtype} {tuple(ids.shape)}")
    if scale is not None and (scale.dtype != torch.float32 or tuple(scale.shape) != (pool,)):
        raise ValueError(f"scale must be float32 [{pool}], got {scale.dtype} {tuple(scale.shape)}")
    if pool == 0 or not 1 <= rank <= MAX_RANK or K == 0 or K % 8 or N == 0:
        raise ValueError(f"{pool} adapters of rank {rank} (1 .. {MAX_RANK}) for K = {K} (a multiple of 8) and N = {N}")
    for name, t in (("y", y), ("a", a), ("b", b), ("ids", ids), ("scale", scale), ("out", out)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if scale is not None and scale.requires_grad:
        raise ValueError("scale has no gradient here: fold it into b to train it")
    if out is not None and (out.dtype != y.dtype or out.shape != y.shape or (rows and (out.stride(1) != 1 and N > 1 or rows > 1 and out.stride(0) < N))):
        raise ValueError(f"out must match y in shape and type, with unit column stride, got {out.dtype} {tuple(out.shape)} strides {out.stride()}")
    return rows, K, N, rank, pool


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows of unit column stride that do not overlap; a copy where they are not."""
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _launch(device: torch.device, call) -> None:
    if device.index == torch.cuda.current_device():
        rc = call(ops._stream())
    else:
        with torch.cuda.device(device):
            rc = call(ops._stream())
    if rc:
        _lib.check(rc)


def _forward(sizes, y, x, a, b, ids, scale, out) -> torch.Tensor:
    """Writes out, returns the hidden vectors."""
    rows, K, N, rank, pool = sizes
    lib = _lib.load()
    hidden = torch.empty(int(lib.wb200_adapters_hidden_bytes(rows, rank, _OUT_CODE[y.dtype])), dtype=torch.uint8, device=x.device)
    _launch(x.device, lambda stream: lib.wb200_adapters_forward(
        rows, K, N, rank, pool, x.data_ptr(), _pitch(x), a.data_ptr(), b.data_ptr(), ids.data_ptr(), int(ids.dtype == torch.int64),
        scale.data_ptr() if scale is not None else None, y.data_ptr(), _pitch(y), out.data_ptr(), _pitch(out), _OUT_CODE[out.dtype],
        hidden.data_ptr(), hidden.numel(), stream))
    return hidden


class _Adapters(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, ids, scale, sizes):
        x, a, b, ids = _rows(x), a.contiguous(), b.contiguous(), ids.contiguous()
        scale = scale.contiguous() if scale is not None else None
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        hidden = _forward(sizes, _rows(y), x, a, b, ids, scale, out)
        ctx.save_for_backward(x, a, b, ids, scale, hidden)
        ctx.sizes = sizes
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, a, b, ids, scale, hidden = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device) if need[1] else None
        da, db = _backward(ctx.sizes, x, a, b, ids, scale, _rows(g), hidden, dx, False, need[2], need[3])
        return (g if need[0] else None), dx, da, db, None, None, None


def _backward(sizes, x, a, b, ids, scale, g, hidden, dx, accumulate: bool, need_a: bool, need_b: bool):
    """Writes dx (or with `accumulate` adds to it), if it is given, and returns the gradients of a and b that are asked for."""
    rows, K, N, rank, pool = sizes
    da = torch.empty_like(a) if need_a else None
    db = torch.empty_like(b) if need_b else None
    if dx is None and not need_a and not need_b:
        return da, db
    lib = _lib.load()
    nbytes = int(lib.wb200_adapters_backward_workspace_bytes(rows, N, rank))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    _launch(x.device, lambda stream: lib.wb200_adapters_backward(
        rows, K, N, rank, pool, x.data_ptr(), _pitch(x), a.data_ptr(), b.data_ptr(), ids.data_ptr(), int(ids.dtype == torch.int64), ptr(scale),
        g.data_ptr(), _pitch(g), hidden.data_ptr(), hidden.numel(), ptr(dx), K, int(accumulate), ptr(da), ptr(db), ws.data_ptr(), nbytes, stream))
    return da, db


class AdaptedLinear(torch.autograd.Function):
    """A frozen layer with adapters as one node: x [rows, K], the adapters' part written onto the layer's output, and onto the layer's part of the
    gradient of x."""

    @staticmethod
    def forward(ctx, x, a, b, ids, scale, layer):
        y = layer._base(x)
        sizes = _check(y, x, a, b, ids, scale, None)
        if y.dtype != torch.bfloat16 or sizes[4] > MAX_TRAINED:
            raise ValueError(f"gradients need a bfloat16 output and at most {MAX_TRAINED} adapters, got {y.dtype} and {sizes[4]}")
        x, a, b, ids = _rows(x), a.contiguous(), b.contiguous(), ids.contiguous()
        scale = scale.contiguous() if scale is not None else None
        hidden = _forward(sizes, y, x, a, b, ids, scale, y)
        ctx.save_for_backward(x, a, b, ids, scale, hidden, layer.weight_codes, layer.weight_scales)
        ctx.sizes = sizes
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, a, b, ids, scale, hidden, codes, scales = ctx.saved_tensors
        g = _rows(g)
        dx = ops.mxfp4_input_grad(g, codes, scales) if ctx.needs_input_grad[0] else None
        da, db = _backward(ctx.sizes, x, a, b, ids, scale, g, hidden, dx, True, *ctx.needs_input_grad[1:3])
        return dx, da, db, None, None, None


def apply_adapters(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, scale: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """y[t] + scale[l] * b[l] @ (a[l] @ x[t]) with l = ids[t], on the current stream.

    y [rows, N] f32 or bf16, x [rows, K] bf16, a [adapters, rank, K] and b [adapters, N, rank] bf16 (adapters of a lower rank are padded
    with zeros), ids [rows] int32 or int64, scale [adapters] f32 or None for ones. A row whose id is outside [0, adapters) has no adapter:
    its y comes back. The sum is made in f32 and rounded once to y's type. out: where to write (y itself, or memory that does not overlap it), not together
    with gradients. Differentiable in y, x, a and b for a bf16 y and pools of at most 65535 adapters; sums over rows are made in a fixed order.
    Limits: rank 256, K a multiple of 8, 4000000 rows, N + K of some 8.3 million, rows of y and out less than 2^24 elements apart.
    """
    native = _lib.native_calls()
    if native is not None and _lib.unwatched("wb200_adapters_forward", "wb200_adapters_backward"):
        result = native.adapters(y, x, a, b, ids, scale, out)
        if result is not None:
            return result if out is None else out
    sizes = _check(y, x, a, b, ids, scale, out)
    rows = sizes[0]
    if torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad):
        if out is not None:
            raise ValueError("out is not taken together with gradients")
        if y.dtype != torch.bfloat16 or sizes[4] > MAX_TRAINED:
            raise ValueError(f"gradients need a bfloat16 y and at most {MAX_TRAINED} adapters, got {y.dtype} and {sizes[4]}")
        if rows == 0:
            return y + 0 * (x.sum() + a.sum() + b.sum())
        return _Adapters.apply(y, x, a, b, ids, scale, sizes)
    if out is None:
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    elif torch.is_grad_enabled() and out.requires_grad:
        raise ValueError("out is not taken together with gradients")
    else:
        ops.written(out)
    if rows:
        _forward(sizes, _rows(y), _rows(x), a.contiguous(), b.contiguous(), ids.contiguous(), scale.contiguous() if scale is not None else None, out)
    return out


class LowRankAdapters(torch.nn.Module):
    """A pool of adapters for one projection: a [adapters, rank, K], b [adapters, N, rank] (bf16), scale [adapters] f32 or None. Given to
    `MXFP4Linear.forward` with the adapter of every row. a and b are parameters; they are trained if `trainable`."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | None = None, trainable: bool = False):
        super().__init__()
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"a must be [adapters, rank, K] and b [adapters, N, rank], got {tuple(a.shape)} and {tuple(b.shape)}")
        self.a = torch.nn.Parameter(a, requires_grad=trainable)
        self.b = torch.nn.Parameter(b, requires_grad=trainable)
        self.register_buffer("scale", scale)

    def forward(self, y: torch.Tensor, x: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        return apply_adapters(y, x, self.a, self.b, ids, self.scale, out)
