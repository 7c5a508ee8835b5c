"""The norms around an encoder block, fused with its gate and residual scale.

    b = branch / rms(branch) * branch_weight
    r = residual + residual_scale * silu(gate) * b
    n = r / rms(r) * next_weight                rms(v) = sqrt(mean(v^2) + eps)

r is the residual stream after the block and n the next block's input.
Statistics and sums are float32; r and n are rounded once.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .packed import PackedActivation


class _BlockNorm(torch.autograd.Function):
    """Inputs branch .. residual_scale are None for the norm alone.  Keeps the
    inputs and two statistics a position; the backward recomputes r."""

    @staticmethod
    def forward(ctx, residual, branch, gate, branch_weight, residual_scale, next_weight, weights,
                lengths, eps, pack):
        # weights: the three as contiguous float32, what the kernels read
        out, normed, stats, codes, scales = _lib.block_norm_forward(
            residual, branch, gate, *weights, lengths, eps, want_statistics=True, pack=pack)
        ctx.save_for_backward(residual, branch, gate, *weights, lengths, stats)
        ctx.eps = eps
        ctx.weight_dtypes = [None if w is None else w.dtype
                             for w in (branch_weight, residual_scale, next_weight)]
        ctx.set_materialize_grads(False)
        if pack:
            ctx.mark_non_differentiable(codes, scales)
        return out, normed, codes, scales

    @staticmethod
    @_lib.first_order
    def backward(ctx, grad_out, grad_normed, _codes, _scales):
        residual, branch, gate, w1, scale, w2, lengths, stats = ctx.saved_tensors
        if grad_out is not None:
            grad_out = _lib.activation(grad_out, "grad_residual", like=residual)
        if grad_normed is not None:
            grad_normed = _lib.activation(grad_normed, "grad_normed", like=residual)
        gr, gb, gg, gw = _lib.block_norm_backward(residual, branch, gate, w1, scale, w2, lengths,
                                                  ctx.eps, stats, grad_out, grad_normed)
        grads = [None if dt is None else g if dt == torch.float32 else g.to(dt)
                 for g, dt in zip(gw.unbind(0), ctx.weight_dtypes)]
        return gr, gb, gg, *grads, None, None, None, None


def _call(residual, branch, gate, branch_weight, residual_scale, next_weight, lengths, eps, pack):
    residual = _lib.activation(residual, "residual" if branch is not None else "x")
    B, T, D = residual.shape
    dev = residual.device
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if branch is not None:
        branch = _lib.activation(branch, "branch", like=residual)
        gate = _lib.activation(gate, "gate", like=residual)
        w1 = _lib.float_vector(branch_weight, "branch_weight", (D,), dev)
        scale = _lib.float_vector(residual_scale, "residual_scale", (D,), dev)
    else:
        w1 = scale = None
    w2 = _lib.float_vector(next_weight, "next_weight" if branch is not None else "weight", (D,),
                           dev)
    lengths = _lib.valid_lengths(lengths, B, T, dev)
    given = (residual, branch, gate, branch_weight, residual_scale, next_weight)
    if _lib.recorded(*given):
        out, normed, codes, scales = _BlockNorm.apply(*given, (w1, scale, w2), lengths, eps,
                                                       bool(pack))
    else:
        out, normed, _, codes, scales = _lib.block_norm_forward(
            residual, branch, gate, w1, scale, w2, lengths, eps, want_statistics=False, pack=pack)
    packed = PackedActivation(codes, scales, D, residual.dtype) if pack else None
    return out, normed, packed


def gated_residual_norm(
    residual: torch.Tensor,
    branch: torch.Tensor,
    gate: torch.Tensor,
    branch_weight: torch.Tensor,
    residual_scale: torch.Tensor,
    next_weight: torch.Tensor,
    lengths: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    pack: bool = False,
):
    """Close one block and open the next: returns (r, n), or with ``pack``
    (r, n, PackedActivation of n), the checkpoint that ``packed_linear`` takes.

    residual, branch, gate: (batch, T, D) of one type, channels contiguous,
    D <= 8192; the weights (D,).  Positions past ``lengths`` give zeros and get
    zero gradients, whatever they hold.  Differentiable in all six tensors;
    weight gradients are summed in a fixed order.
    """
    if branch is None or gate is None:
        raise ValueError("branch and gate are required (rms_norm is the norm alone)")
    out, normed, packed = _call(residual, branch, gate, branch_weight, residual_scale, next_weight,
                                lengths, eps, pack)
    return (out, normed, packed) if pack else (out, normed)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, lengths: Optional[torch.Tensor] = None,
             eps: float = 1e-6, pack: bool = False):
    """n = x / rms(x) * weight, the norm before the first block: n, or with
    ``pack`` (n, PackedActivation of n).  Same rules as gated_residual_norm."""
    _, normed, packed = _call(x, None, None, None, None, weight, lengths, eps, pack)
    return (normed, packed) if pack else normed
