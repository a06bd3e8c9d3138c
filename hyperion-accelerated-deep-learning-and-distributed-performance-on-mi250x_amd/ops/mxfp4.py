"""Microscaled 4-bit floating point (MXFP4): quantisation and linear layers with a frozen 4-bit weight.

A LoRA fine-tune never changes its base weights, and at a few hundred tokens it is the time to stream
them (:mod:`.linear`): in 4 bits they take 17/64 of the bf16 bytes, in memory and on the way to the
matrix cores.  32 consecutive elements of a row share a power-of-two scale (one byte, e8m0); an element
is one of 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign (e2m1), two to a byte, the first in the low half
(``csrc/kernels/mxfp4.hip``).  Rows that are no multiple of 32 long are padded with zeros.

* :func:`quantize_mxfp4` rounds to the nearest value (ties to even) under the scale ``2^(floor(log2(max
  |x|)) - 2)`` of each block; magnitudes above 6 of it become 6.  A block with a NaN or an infinity is NaN.
* :func:`mxfp4_linear` is ``x Wᵀ (+ b)`` and, in the backward, ``dy W``: a 4-bit value is a bf16 number
  exactly, so the products run on the bf16 matrix instructions with fp32 sums.  fp16 and fp32
  activations are split into two or three bf16 numbers whose sum they are, and lose nothing either.
  The weight is frozen: it has no gradient.

The products decode the codes on their way to the matrix instructions, in one launch (fp16 and fp32 activations are
split by another); the largest, where it is faster, decode the weight to bf16 once (a buffer of the call) and run on the
tiled GEMM.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _native
from .linear import bias_grad

BLOCK = 32
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class MXFP4Tensor:
    """Rows of 4-bit values: ``codes`` uint8 [R, 16 nb], ``scales`` uint8 [R, nb], nb = ceil(K / 32), of a
    tensor of ``shape`` [..., K] with R rows."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: Tuple[int, ...]):
        shape = tuple(int(n) for n in shape)
        if len(shape) < 1 or any(n < 0 for n in shape):
            raise ValueError(f"MXFP4Tensor: shape must be [..., K], got {shape}")
        nb, rows = -(-shape[-1] // BLOCK), math.prod(shape[:-1])
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"MXFP4Tensor: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
        if codes.shape != (rows, 16 * nb) or scales.shape != (rows, nb):
            raise ValueError(f"MXFP4Tensor: shape {shape} needs codes {(rows, 16 * nb)} and scales {(rows, nb)}, "
                             f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"MXFP4Tensor: codes on {codes.device}, scales on {scales.device}")
        self.codes, self.scales, self.shape = codes.contiguous(), scales.contiguous(), shape
        if self.codes.data_ptr() % 16:
            self.codes = self.codes.clone()  # the kernels read 16 bytes at a time
        if self.scales.data_ptr() % 4:
            self.scales = self.scales.clone()  # and four scales

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={self.shape}, device='{self.device}')"

    def _rows(self, dtype: torch.dtype, cols: int) -> torch.Tensor:
        """[R, cols] values; cols is K, or 32 nb with the padding."""
        if _native.use_native(self.codes, op="mxfp4"):
            return _native.native().mx_dequantize(self.codes, self.scales, cols, dtype)
        return _decode_reference(self.codes, self.scales)[:, :cols].to(dtype)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values in ``dtype`` (exact in bf16 and fp32 down to their smallest numbers; fp16 rounds once)."""
        if dtype not in _native.DTYPE_CODE:
            raise TypeError(f"MXFP4Tensor.dequantize: fp32, bf16 or fp16, got {dtype}")
        return self._rows(dtype, self.shape[-1]).view(self.shape)


def _decode_reference(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """PyTorch oracle of the decoding: [R, 32 nb] in fp32."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    q = torch.stack([codes & 15, codes >> 4], dim=-1).view(codes.shape[0], scales.shape[1], BLOCK)
    s = torch.exp2(scales.double() - 127.0).float()
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (table[q.long()] * s[..., None]).view(codes.shape[0], 2 * codes.shape[1])


def _encode_reference(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """PyTorch oracle of mx_quantize over [R, K]."""
    R, K = x.shape
    nb = -(-K // BLOCK)
    x = F.pad(x.float(), (0, -K % BLOCK)).view(R, nb, BLOCK)
    amax = x.abs().amax(dim=2, keepdim=True)
    bad = ~torch.isfinite(amax)
    e = (torch.frexp(torch.where(bad, torch.ones_like(amax), amax))[1] - 3).clamp(min=-127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    a = x.abs().double() * torch.exp2(-e.double())
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).nan_to_num(0.0).to(torch.uint8)
    code = (code | (torch.signbit(x).to(torch.uint8) << 3)).view(R, 16 * nb, 2)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code[..., 0] | (code[..., 1] << 4), scale[..., 0]


def quantize_mxfp4(x: torch.Tensor) -> MXFP4Tensor:
    """``x`` [..., K] (fp32, bf16 or fp16) in blocks of 32 along its last dimension."""
    if x.dtype not in _native.DTYPE_CODE:
        raise TypeError(f"quantize_mxfp4: x must be fp32, bf16 or fp16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("quantize_mxfp4: x must be [..., K]")
    x = x.detach()
    K = x.shape[-1]
    rows = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), K)
    if K > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    if _native.use_native(rows, op="mxfp4"):
        _native.count("mxfp4_quantize")
        codes, scales = _native.native().mx_quantize(rows)
    else:
        codes, scales = _encode_reference(rows)
    return MXFP4Tensor(codes, scales, tuple(x.shape))


def _unit_rows(x: torch.Tensor, n: int) -> torch.Tensor:
    """[M, n] with unit column stride (a view where it is one)."""
    x2 = x if x.dim() == 2 else x.reshape(-1, n)
    return x2 if n <= 1 or x2.stride(1) == 1 else x2.contiguous()


def _bias32(bias: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if bias is None:
        return None
    b = bias.detach().float().contiguous()
    return b if b.data_ptr() % 16 == 0 else b.clone()


class _MXLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, w):
        N, K = w.shape
        native = _native.use_native(x, w.codes, op="mxfp4")
        if x.numel() == 0 or N == 0:
            y = x.new_zeros(*x.shape[:-1], N) + (0 if bias is None else bias.to(x.dtype))
        elif native:
            _native.count("mxfp4_linear")
            y = _native.native().mx_linear(_unit_rows(x, K), w.codes, w.scales, _bias32(bias))
        else:
            y = x.float() @ w._rows(torch.float32, K).t()
            y = (y if bias is None else y + bias.float()).to(x.dtype)
        if ctx.needs_input_grad[0]:
            ctx.weight = None
            if w.codes.is_inference() or w.scales.is_inference():  # (these have no version to check, and cannot be saved)
                ctx.weight = w.codes, w.scales
            else:
                ctx.save_for_backward(w.codes, w.scales)  # (a weight loaded before the backward is noticed there)
        ctx.wshape, ctx.native, ctx.xshape, ctx.bdtype = w.shape, native, x.shape, None if bias is None else bias.dtype
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        N, K = ctx.wshape
        dx = db = None
        if ctx.needs_input_grad[0]:
            codes, scales = ctx.weight or ctx.saved_tensors
            if dy.numel() == 0 or K == 0:
                dx = dy.new_zeros(ctx.xshape)
            elif ctx.native:
                _native.count("mxfp4_dgrad")
                dx = _native.native().mx_linear_dgrad(_unit_rows(dy, N), codes, scales, K).view(ctx.xshape)
            else:
                dx = (dy.float() @ _decode_reference(codes, scales)[:, :K]).to(dy.dtype)
        if ctx.bdtype is not None and ctx.needs_input_grad[1]:
            db = bias_grad(dy.reshape(math.prod(dy.shape[:-1]), N).contiguous(), ctx.bdtype)
        return dx, db, None


def mxfp4_linear(x: torch.Tensor, weight: MXFP4Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x Wᵀ (+ bias)`` with a frozen 4-bit ``weight`` of shape [N, K]; differentiable (once) in x and bias.
    Under autocast x is cast to the autocast dtype first, like a linear layer's."""
    if not isinstance(weight, MXFP4Tensor) or len(weight.shape) != 2:
        raise TypeError("mxfp4_linear: weight must be an MXFP4Tensor of shape [N, K]")
    if torch.is_autocast_enabled(x.device.type):
        x = x.to(torch.get_autocast_dtype(x.device.type))
    if x.dtype not in _native.DTYPE_CODE:
        raise TypeError(f"mxfp4_linear: x must be fp32, bf16 or fp16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"mxfp4_linear: x {tuple(x.shape)} does not match weight {weight.shape}")
    if x.device != weight.device or (bias is not None and bias.device != x.device):
        raise ValueError("mxfp4_linear: x, weight and bias must be on one device")
    if bias is not None and (bias.shape != (weight.shape[0],) or not bias.is_floating_point()):
        raise ValueError(f"mxfp4_linear: bias must be a floating [{weight.shape[0]}], got {tuple(bias.shape)} {bias.dtype}")
    needs_grad = x.requires_grad or (bias is not None and bias.requires_grad)
    return _native.apply_fn(_MXLinearFn, x, bias, weight, needs_grad=needs_grad)


class MXFP4Linear(nn.Module):
    """A linear layer whose weight is frozen in 4 bits (buffers ``weight_codes`` / ``weight_scales``)."""

    frozen_buffers = ("weight_codes", "weight_scales")  # data parallelism need not keep them in step

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        nb = -(-in_features // BLOCK)
        self.register_buffer("weight_codes", torch.zeros(out_features, 16 * nb, dtype=torch.uint8, device=device))
        self.register_buffer("weight_scales", torch.zeros(out_features, nb, dtype=torch.uint8, device=device))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device)) if bias else None

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "MXFP4Linear":
        """The layer with ``linear``'s weight quantised; its bias is kept (the same parameter)."""
        m = cls(linear.in_features, linear.out_features, bias=False, device="meta")
        q = quantize_mxfp4(linear.weight)
        m.weight_codes, m.weight_scales, m.bias = q.codes, q.scales, linear.bias
        return m

    @property
    def weight(self) -> MXFP4Tensor:
        return MXFP4Tensor(self.weight_codes, self.weight_scales, (self.out_features, self.in_features))

    def forward(self, x: torch.Tensor, link=None, blink=None) -> torch.Tensor:
        """``link`` / ``blink``: the gradient links of ``ops.linear.Linear``, which stay unarmed here."""
        return mxfp4_linear(x, self.weight, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
