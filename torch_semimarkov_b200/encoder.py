"""A gated recurrent encoder in front of the CRF head.

Each block reads the normed residual stream, projects it to a value, a forget
gate and an output gate, runs the gated linear recurrence over time, and adds
the recurrence's output, normed, gated and scaled, to the stream:

    v, f, o = n W^T + b
    h = gated_linear_recurrence(v, f)
    r, n = gated_residual_norm(r, h, o, ...)

With ``bidirectional`` every second block scans backwards in time.  n is kept
for W's gradient in 8 bits (``checkpoint_8bit``).

    encoder = GatedRecurrentEncoder(input_dim, 512, num_layers=4).cuda()
    head = SemiMarkovCRFHead(num_classes, max_duration, hidden_dim=512).cuda()
    loss = head.compute_loss(encoder(features, lengths).float(), lengths, labels)
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from . import _lib
from .block_norm import gated_residual_norm, rms_norm
from .packed import packed_linear
from .recurrence import gated_linear_recurrence, gated_linear_recurrence_step


class GatedRecurrentEncoder(nn.Module):
    """Sequence encoder of gated linear recurrences.

    Args:
        input_dim: features per position.
        hidden_dim: width D of the residual stream (at most 8192).
        num_layers: number of blocks.
        bidirectional: odd blocks scan from the end of each sequence.
        checkpoint_8bit: keep the projections' inputs in 8 bits for the
            backward.
        dtype: type of the activations (parameters stay as they are made,
            float32); float32, bfloat16 or float16.
        eps: of the norms.
    """

    def __init__(self, input_dim: int, hidden_dim: int, num_layers: int = 2,
                 bidirectional: bool = True, checkpoint_8bit: bool = True,
                 dtype: torch.dtype = torch.bfloat16, eps: float = 1e-6):
        super().__init__()
        if num_layers < 1:
            raise ValueError(f"num_layers must be >= 1, got {num_layers}")
        if dtype not in _lib.ACTIVATION_DTYPES:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        D = hidden_dim
        self.hidden_dim = D
        self.num_layers = num_layers
        self.bidirectional = bidirectional
        self.checkpoint_8bit = checkpoint_8bit
        self.dtype = dtype
        self.eps = eps
        self.embed = nn.Linear(input_dim, D)
        self.first_weight = nn.Parameter(torch.ones(D))
        self.in_weight = nn.ParameterList()
        self.in_bias = nn.ParameterList()
        self.branch_weight = nn.ParameterList()
        self.residual_scale = nn.ParameterList()
        self.next_weight = nn.ParameterList()
        # forget gates start with memories from a few to some hundred positions
        memory = torch.linspace(1.0, 6.0, D)
        for _ in range(num_layers):
            self.in_weight.append(nn.Parameter(torch.randn(3 * D, D) * D ** -0.5))
            self.in_bias.append(nn.Parameter(torch.cat([torch.zeros(D), memory, torch.ones(D)])))
            self.branch_weight.append(nn.Parameter(torch.ones(D)))
            self.residual_scale.append(nn.Parameter(torch.full((D,), (2 * num_layers) ** -0.5)))
            self.next_weight.append(nn.Parameter(torch.ones(D)))

    def _project(self, n: Tensor, packed, lengths, layer: int):
        w, b = self.in_weight[layer], self.in_bias[layer]
        if packed is not None:
            p = packed_linear(n, w, b, packed, lengths)
        else:
            p = F.linear(n, w.to(n.dtype), b.to(n.dtype))
        return p.split(self.hidden_dim, dim=-1)

    def forward(self, features: Tensor, lengths: Optional[Tensor] = None) -> Tensor:
        """features (batch, T, input_dim) to hidden states (batch, T, D) of type
        ``dtype``, zeros past each length."""
        x = features.to(self.dtype)
        if lengths is not None:
            B, T = x.shape[:2]
            lengths = _lib.valid_lengths(lengths, B, T, x.device)
            if torch.is_grad_enabled():
                # the embedding's weight gradient is a product over all positions,
                # and a zero gradient times what padding may hold need not be zero
                padding = torch.arange(T, device=x.device) >= lengths[:, None]
                x = x.masked_fill(padding[..., None], 0.0)
        r = F.linear(x, self.embed.weight.to(x.dtype), self.embed.bias.to(x.dtype))
        pack = self.checkpoint_8bit and torch.is_grad_enabled()
        packed = None
        n = rms_norm(r, self.first_weight, lengths, self.eps, pack)
        if pack:
            n, packed = n
        for k in range(self.num_layers):
            v, f, o = self._project(n, packed, lengths, k)
            h, _ = gated_linear_recurrence(v, f, lengths=lengths,
                                           reverse=self.bidirectional and k % 2 == 1)
            last = k + 1 == self.num_layers
            out = gated_residual_norm(r, h, o, self.branch_weight[k], self.residual_scale[k],
                                      self.next_weight[k], lengths, self.eps, pack and not last)
            r, n = out[:2]
            packed = out[2] if pack and not last else None
        return n

    def initial_states(self, batch: int) -> list[Tensor]:
        """Zero states for ``step``: one (batch, D) float32 tensor a block."""
        dev = self.first_weight.device
        return [torch.zeros(batch, self.hidden_dim, device=dev) for _ in range(self.num_layers)]

    @torch.no_grad()
    def step(self, features: Tensor, states: list[Tensor]) -> Tensor:
        """One position of ``batch`` streams (serving): features (batch,
        input_dim) to hidden states (batch, D).  ``states`` are updated in
        place.  Not for a bidirectional encoder, which needs the future."""
        if self.bidirectional:
            raise ValueError("step needs an encoder with bidirectional=False")
        if len(states) != self.num_layers:
            raise ValueError(f"states must hold {self.num_layers} tensors")
        x = features.to(self.dtype)[:, None]
        r = F.linear(x, self.embed.weight.to(x.dtype), self.embed.bias.to(x.dtype))
        n = rms_norm(r, self.first_weight, eps=self.eps)
        for k in range(self.num_layers):
            v, f, o = self._project(n, None, None, k)
            h, _ = gated_linear_recurrence_step(v[:, 0], f[:, 0], states[k], out_state=states[k])
            r, n = gated_residual_norm(r, h[:, None], o, self.branch_weight[k],
                                       self.residual_scale[k], self.next_weight[k], eps=self.eps)
        return n[:, 0]
