"""8-bit activation checkpoints, and the linear layer whose backward uses them.

What a linear layer keeps for its weight gradient is its input.  Here that
input is kept in 8 bits: 32 neighbouring channels of a position share the
smallest power of two 2^e with max |x| <= 127 * 2^e, and are stored as int8
codes rint(x / 2^e).  The backward's weight gradient reads the codes directly.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib


@dataclass
class PackedActivation:
    """An activation (batch, time, channels) stored in 8 bits.

    codes (batch, time, 32 * ceil(channels / 32)) int8, zero past the last
    channel; scales (batch, time, ceil(channels / 32)) uint8, e + 127 (0: a
    group of zeros, 255: a group that held a value that was not finite, which
    reads back as NaN)."""

    codes: torch.Tensor
    scales: torch.Tensor
    channels: int
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:2], self.channels))

    def unpack(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The stored values, in the type they were packed from or ``dtype``."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _lib.ACTIVATION_DTYPES:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        _check(self)
        return _lib.unpack(self.codes, self.scales, self.channels, dtype)


def _check(p: PackedActivation):
    if not isinstance(p, PackedActivation):
        raise ValueError("packed must be a PackedActivation")
    G = -(-p.channels // _lib.PACK_GROUP)
    if (p.codes.dim() != 3 or p.codes.dtype != torch.int8 or p.scales.dtype != torch.uint8
            or p.codes.shape[2] != G * _lib.PACK_GROUP
            or p.scales.shape != (*p.codes.shape[:2], G)
            or not p.codes.is_contiguous() or not p.scales.is_contiguous()
            or p.codes.device != p.scales.device):
        raise ValueError("codes and scales do not have a packed activation's layout")
    if not p.codes.is_cuda:
        raise RuntimeError("torch_semimarkov_b200 runs on CUDA devices only (the packed "
                           "activation is on the CPU)")


def pack_activation(x: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> PackedActivation:
    """Store x (batch, T, channels) in 8 bits.  Positions past a sequence's
    length are stored as zeros, whatever they hold.  No gradient passes through a
    checkpoint: what is read back stands apart from x."""
    x = _lib.activation(x, "x")
    _lib.refuse_tangents("pack_activation", x)
    lengths = _lib.valid_lengths(lengths, x.shape[0], x.shape[1], x.device)
    codes, scales = _lib.pack(x, lengths)
    return PackedActivation(codes, scales, x.shape[2], x.dtype)


def packed_weight_grad(grad_output: torch.Tensor, packed: PackedActivation,
                       lengths: Optional[torch.Tensor] = None,
                       dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Weight gradient of y = x W^T from x's checkpoint: the (M, channels) sum
    over valid positions of grad_output (batch, T, M)^T x, summed in float32
    and returned as ``dtype`` (grad_output's type if None).  The result is not
    differentiable."""
    _check(packed)
    grad_output = _lib.activation(grad_output, "grad_output")
    _lib.refuse_tangents("packed_weight_grad", grad_output)
    B, T, _ = grad_output.shape
    if packed.codes.shape[:2] != (B, T) or packed.codes.device != grad_output.device:
        raise ValueError(f"packed holds {tuple(packed.shape)} on {packed.codes.device}, "
                         f"grad_output is {tuple(grad_output.shape)} on {grad_output.device}")
    dtype = grad_output.dtype if dtype is None else dtype
    if dtype not in _lib.ACTIVATION_DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    lengths = _lib.valid_lengths(lengths, B, T, grad_output.device)
    return _lib.packed_weight_grad(grad_output, packed.codes, packed.scales, packed.channels,
                                   packed.dtype, lengths, dtype)


def _linear(x, weight, bias):
    """x weight^T + bias in x's type: one product whose sums take the bias before
    they are rounded."""
    w = weight.to(x.dtype)
    if bias is None:
        return torch.matmul(x, w.t())
    B, T, D = x.shape
    return torch.addmm(bias.to(x.dtype), x.reshape(B * T, D), w.t()).view(B, T, w.shape[0])


class _PackedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, packed, lengths):
        y = _linear(x, weight, bias)
        ctx.save_for_backward(weight, packed.codes, packed.scales, lengths)
        ctx.packed_dtype = packed.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, grad):
        weight, codes, scales, lengths = ctx.saved_tensors
        grad = _lib.activation(grad, "grad_output")
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = torch.matmul(grad, weight.to(grad.dtype))
        if ctx.needs_input_grad[1]:
            gw = _lib.packed_weight_grad(grad, codes, scales, weight.shape[1], ctx.packed_dtype,
                                         lengths, weight.dtype)
        if ctx.needs_input_grad[2]:
            if lengths is not None:
                T = grad.shape[1]
                live = torch.arange(T, device=grad.device) < lengths[:, None]
                grad = grad.masked_fill(~live[..., None], 0.0)
            gb = grad.sum((0, 1), dtype=torch.float32).to(ctx.bias_dtype)
        return gx, gw, gb, None, None


def packed_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  packed: Optional[PackedActivation] = None,
                  lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x weight^T + bias that keeps x in 8 bits for its weight gradient.

    x (batch, T, D); weight (M, D) and bias (M,) in x's type or float32;
    ``packed``: x's checkpoint where it is at hand (``gated_residual_norm``
    and ``rms_norm`` write it beside their result), else it is made here.
    Positions past ``lengths`` add nothing to the gradients of weight and bias.
    The gradient of x is exact; the weight's is that of the stored values.
    """
    x = _lib.activation(x, "x")
    B, T, D = x.shape
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] != D:
        raise ValueError(f"weight must be a (M, {D}) tensor")
    if weight.dtype not in _lib.ACTIVATION_DTYPES or weight.device != x.device:
        raise ValueError(f"weight must be float32, bfloat16 or float16 on {x.device}")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.device != x.device):
        raise ValueError(f"bias must have shape ({weight.shape[0]},) on {x.device}")
    lengths = _lib.valid_lengths(lengths, B, T, x.device)
    needs = torch.is_grad_enabled() and (weight.requires_grad or x.requires_grad
                                         or (bias is not None and bias.requires_grad))
    if not needs:
        return _linear(x, weight, bias)
    if packed is None:
        packed = pack_activation(x, lengths)
    else:
        _check(packed)
        if packed.shape != x.shape or packed.codes.device != x.device:
            raise ValueError(f"packed holds {tuple(packed.shape)}, x is {tuple(x.shape)}")
    return _PackedLinear.apply(x, weight, bias, packed, lengths)
