"""Gated linear recurrence: the sequence mixer of a recurrent encoder.

    f_t = sigmoid(gate_t)
    state_t = f_t * state_{t-1} + (1 - f_t) * x_t,    h_t = state_t

over each sequence's valid positions, channel by channel, ascending or (the
other half of a bidirectional encoder) descending in t.  The scan over time is
parallel; states and sums are float32, and ``h`` is rounded once.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib


class _GatedLinearRecurrence(torch.autograd.Function):
    """Keeps x, gate and the float32 state at the start of each run of
    positions; the backward recomputes the states inside a run from those."""

    @staticmethod
    def forward(ctx, x, gate, initial_state, start, lengths, reverse):
        # start holds initial_state as contiguous float32, what the kernels read
        h, state, saved = _lib.recurrence_forward(x, gate, start[0], lengths, reverse,
                                                  want_saved=True)
        ctx.save_for_backward(x, gate, lengths, saved)
        ctx.reverse = reverse
        ctx.initial_dtype = None if initial_state is None else initial_state.dtype
        ctx.set_materialize_grads(False)
        return h, state

    @staticmethod
    @_lib.first_order
    def backward(ctx, grad_h, grad_state):
        x, gate, lengths, saved = ctx.saved_tensors
        if grad_h is not None:
            grad_h = _lib.activation(grad_h, "grad_h", like=x)
        if grad_state is not None:
            grad_state = grad_state.to(torch.float32).contiguous()
        want = ctx.initial_dtype is not None and ctx.needs_input_grad[2]
        gx, gg, gi = _lib.recurrence_backward(x, gate, lengths, ctx.reverse, saved, grad_h,
                                              grad_state, want)
        if want and ctx.initial_dtype != torch.float32:
            gi = gi.to(ctx.initial_dtype)
        return gx, gg, gi, None, None, None


def gated_linear_recurrence(
    x: torch.Tensor,
    gate: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
    reverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Run the recurrence over (batch, time, channel) inputs.

    Args:
        x, gate: (batch, T, D) float32, bfloat16 or float16, of one type.
            Channels contiguous, other strides free: slices of one wider
            projection are read in place.
        initial_state: (batch, D), zeros if None.
        lengths: (batch,) valid positions of each sequence, all if None.
            Positions past a length give h = 0, leave the state alone and get
            zero gradients, whatever they hold.
        reverse: scan from the last valid position to the first.

    Returns (h (batch, T, D) of x's type, final_state (batch, D) float32, the
    state after the last position scanned).  Differentiable in x, gate and
    initial_state.
    """
    x = _lib.activation(x, "x")
    gate = _lib.activation(gate, "gate", like=x)
    B, T, D = x.shape
    lengths = _lib.valid_lengths(lengths, B, T, x.device)
    s0 = None
    if initial_state is not None:
        s0 = _lib.float_vector(initial_state, "initial_state", (B, D), x.device)
    if _lib.recorded(x, gate, initial_state):
        return _GatedLinearRecurrence.apply(x, gate, initial_state, (s0,), lengths, bool(reverse))
    h, state, _ = _lib.recurrence_forward(x, gate, s0, lengths, reverse, want_saved=False)
    return h, state


def gated_linear_recurrence_step(
    x: torch.Tensor,
    gate: torch.Tensor,
    state: torch.Tensor,
    active: Optional[torch.Tensor] = None,
    out_state: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One position of ``batch`` independent streams (serving).

    Args:
        x, gate: (batch, D) of one activation type, channels contiguous.
        state: (batch, D) float32, the streams' states.
        active: (batch,) bool; a stream that is not active keeps its state and
            gives h = 0.  All are active if None.
        out_state: where the new state goes; pass ``state`` itself to update
            it in place.  A new tensor if None.

    Returns (h (batch, D) of x's type, the new state).  No gradient.
    """
    for t, name in ((x, "x"), (gate, "gate"), (state, "state")):
        if not isinstance(t, torch.Tensor) or t.dim() != 2:
            raise ValueError(f"{name} must be a (batch, D) tensor")
    dev = x.device
    if not x.is_cuda:
        raise RuntimeError("torch_semimarkov_b200 runs on CUDA devices only (x is on the CPU; "
                           "there is no CPU fallback)")
    if x.dtype not in _lib.ACTIVATION_DTYPES:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if gate.shape != x.shape or gate.dtype != x.dtype or gate.device != dev:
        raise ValueError("gate must have x's shape, type and device")
    if x.shape[1] < 1:
        raise ValueError("x has no channels")
    for t, name in ((state, "state"), (out_state, "out_state")):
        if t is not None and (t.shape != x.shape or t.dtype != torch.float32 or t.device != dev
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 {tuple(x.shape)} tensor on "
                             f"{dev}")
    if active is not None:
        if active.shape != x.shape[:1] or active.dtype != torch.bool or active.device != dev:
            raise ValueError(f"active must be a ({x.shape[0]},) bool tensor on {dev}")
        active = active.contiguous()
    if x.stride(1) != 1:
        x = x.contiguous()
    if gate.stride(1) != 1:
        gate = gate.contiguous()
    _lib.refuse_tangents("gated_linear_recurrence_step", x, gate, state)
    return _lib.recurrence_step(x, gate, state, active, out_state)
