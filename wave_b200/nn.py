"""A linear layer on the MXFP4 path: weights held as packed E2M1 codes with their scales already in
the layout the GEMM reads, activations quantised on the fly.

Counterpart of the reference's module wrappers around its kernels (wave_lang/kernel/wave/nn/linear.py:147
`WaveLinear`, nn/quant_linear.py:196 `WaveQuantLinear`, which is FP8 per-tensor); the reference has
no MXFP4 module. forward(x) = dequant(quantise(x)) @ dequant(W)^T, output bf16 or f32.
"""

from __future__ import annotations

import torch

from . import _lib, ops
from .adapters import AdaptedLinear
from .lang import as_output_dtype


_entry = None  # the function that the host module calls


def _native():
    """The host module, unless it cannot be used or a caller has put something in the place of what it calls, to watch or to redirect calls."""
    global _entry
    if _entry is None and _lib.fast() is not None:
        _entry = _lib._fast_entries["wb200_mxfp4_gemm_quantize_a"]
    lib = _lib._lib
    if not _lib._fast or _lib.load is not _lib._loader or lib is not _lib._fast_lib or lib.wb200_mxfp4_gemm_quantize_a is not _entry:
        return None
    return _lib._fast


_ALONE = object()  # in the place of ids: the layer's own output


class _FrozenLinear(torch.autograd.Function):
    """A layer's output with the gradient of its input; the rounding of the activations to MXFP4 counts as the identity."""

    @staticmethod
    def forward(ctx, x, layer):
        ctx.save_for_backward(layer.weight_codes, layer.weight_scales)
        return layer._base(x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        codes, scales = ctx.saved_tensors
        dx = ops.mxfp4_input_grad(g.reshape(-1, g.shape[-1]), codes, scales)
        return dx.reshape(*g.shape[:-1], dx.shape[1]), None


class MXFP4Linear(torch.nn.Module):
    def __init__(self, weight_codes: torch.Tensor, weight_scales: torch.Tensor, output_dtype=torch.bfloat16, input_grad: bool = False):
        """weight_codes [N, K/2] uint8, weight_scales [N, K/32] uint8 (row-major E8M0), both on the GPU. The GEMM reads the scales in
        packings that are made here, on the current stream, and anew when a state dict is loaded.
        input_grad: gradients flow through the frozen weight to an x that requires one (bf16 x and output); without it the output
        is detached from x."""
        super().__init__()
        ops._as_u8(weight_codes, "weight_codes")
        self.out_features, half_k = weight_codes.shape
        self.in_features = half_k * 2
        self.output_dtype = as_output_dtype(output_dtype).torch_dtype
        if input_grad and self.output_dtype != torch.bfloat16:
            raise ValueError("the input gradient is taken from a bfloat16 output")
        self.input_grad = input_grad
        self.register_buffer("weight_codes", weight_codes.contiguous())
        self.register_buffer("weight_scales", weight_scales.contiguous())
        self._pack()

    input_grad = False

    # Decode calls (at most 128 rows) may read a second packing, per tile of the height h that gives every SM the same number of
    # weight tiles: one height per layer, as it follows from out_features, and 128 / h times the bytes of the usual packing. Made with that one, not
    # by the first call that reads it: other streams' calls would have to wait for that call's.
    _packed = _packed_low = None
    _native_scales = None  # of both, as the native call takes them

    def _pack(self) -> None:
        self._packed = self._pack_as(self._packed, 128)
        h = self._low_rows()
        self._packed_low = None if h == 128 else self._pack_as(self._packed_low, h)
        low = self._packed_low or self._packed
        self._native_scales = self._packed.rows, self._packed.K, self._packed.data, low.data, low.tile_rows

    def _pack_as(self, old: ops.PackedScales | None, tile_rows: int) -> ops.PackedScales:
        """In the memory of the packing that there is, if it is of that form: captured graphs hold its address, as they hold that of the codes,
        which a state dict is copied into."""
        s = self.weight_scales
        same = old is not None and old.device == s.device and (old.rows, old.K, old.tile_rows) == (s.shape[0], s.shape[1] * ops.SCALE_GROUP_SIZE, tile_rows)
        return ops.repack_scales(s, out=old.data if same else None, tile_rows=tile_rows)

    def _low_rows(self) -> int:
        """The height that decode calls of some number of rows read, 128 where none does. (One of each class that
        `ops.decode_tile_rows_for` tells apart: by rows, and by whether rows of the output start on 16 bytes, as that of one row does.)"""
        N, K, device = self.out_features, self.in_features, self.weight_scales.device
        aligned = N * self.output_dtype.itemsize % 16 == 0
        for rows, c_aligned in ((1, True), (2, aligned), (32, aligned), (64, aligned), (128, aligned)):
            h = ops.decode_tile_rows_for(rows, N, K, device, c_aligned=c_aligned)
            if h != 128:
                return h
        return 128

    def _load_from_state_dict(self, *args, **kwargs) -> None:
        super()._load_from_state_dict(*args, **kwargs)
        if self.weight_scales is not None and self.weight_scales.is_cuda:
            self._pack()

    @property
    def _packed_decode(self) -> ops.PackedScales:
        return self._packed if self._packed_low is None else self._packed_low

    @classmethod
    def from_float(cls, weight: torch.Tensor, output_dtype=torch.bfloat16, input_grad: bool = False) -> "MXFP4Linear":
        """Quantise an f32 / bf16 [N, K] weight on the GPU."""
        q, s, _ = ops.quantize_mxfp4(weight, want_rowmajor=True, want_packed=False)
        return cls(q, s, output_dtype, input_grad)

    def forward(self, x: torch.Tensor, adapters=None, ids: torch.Tensor | None = None) -> torch.Tensor:
        """x [..., K] -> [..., N]. adapters: a `LowRankAdapters` pool, ids [...]: the adapter of every row (outside the pool: none); what they
        add is rounded onto the layer's rounded output. They take a bf16 x."""
        if adapters is not None or (self.input_grad and ids is not _ALONE):
            return self._forward_trained(x, adapters, ids)
        # a call whose tensors need no preparation (here, not a function away: it is microseconds long); anything else comes back unhandled
        native, scales = _native(), self._native_scales
        if native is None or scales is None:
            return self._forward_checked(x)
        y = native.linear(x, self._buffers.get("weight_codes"), scales, self.output_dtype, ops._pool._fast or ops._pool.fast)
        if type(y) is int:
            _lib.check(y)
        elif y is not None:
            return y
        return self._forward_checked(x)

    def _forward_trained(self, x: torch.Tensor, adapters, ids) -> torch.Tensor:
        ops.refuse_tangents(x)
        through = torch.is_grad_enabled() and x.requires_grad
        if through:
            if not self.input_grad:
                raise ValueError("the gradient of x needs the layer's part: make the layer with input_grad=True, or pass x.detach()")
            if x.dtype != torch.bfloat16:
                raise ValueError(f"the gradient of x needs a bfloat16 x, got {x.dtype}")
        if adapters is None:
            return _FrozenLinear.apply(x, self) if through else self._base(x)
        if ids is None or ids.shape != x.shape[:-1]:
            raise ValueError(f"ids must hold the adapter of every row of x, {tuple(x.shape[:-1])}")
        x2, ids = x.reshape(-1, self.in_features), ids.reshape(-1)
        if through:
            y = AdaptedLinear.apply(x2, adapters.a, adapters.b, ids, adapters.scale, self)
        else:
            y = self._base(x2)
            trained = torch.is_grad_enabled() and (adapters.a.requires_grad or adapters.b.requires_grad)
            y = adapters(y, x2, ids, out=None if trained else y)
        return y.reshape(*x.shape[:-1], self.out_features)

    def _base(self, x: torch.Tensor) -> torch.Tensor:
        """The layer's own output, without a graph."""
        return MXFP4Linear.forward(self, x, None, _ALONE)

    def _forward_checked(self, x: torch.Tensor) -> torch.Tensor:
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features)
        out = torch.empty(x2.shape[0], self.out_features, dtype=self.output_dtype, device=x.device)
        packed = self._packed
        if x2.shape[0] <= 128:
            packed = self._decode_packing(out)
        ops.quantized_gemm(x2, self.weight_codes, packed, out)
        return out.reshape(*lead, self.out_features)

    def _decode_packing(self, out: torch.Tensor) -> ops.PackedScales:
        low = self._packed_low
        if low is None:
            return self._packed
        h = ops.decode_tile_rows_for(out.shape[0], self.out_features, self.in_features, out.device, c_aligned=ops.rows_aligned(out))
        return low if h == low.tile_rows else self._packed
