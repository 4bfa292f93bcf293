"""Gated linear recurrence: a cheap recurrent mixer beside the delta-rule memory layer.

Per batch row and channel, with a_t = sigmoid(gate_t):

    h_t = a_t h_{t-1} + (1 - a_t) x_t        y_t = h_t silu(out_gate_t)

The state is fp32 whatever the storage type.  ``gated_scan`` and ``gated_scan_packed``
run a sequence and have a backward pass; ``gated_scan_step`` advances a state in place by
one token.  dg_gated_scan_forward / _backward / _step in include/deltagrid_b200.h hold
the exact contract.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import _hsru


def gated_scan(x: torch.Tensor, gate: torch.Tensor, out_gate: Optional[torch.Tensor] = None,
               h0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
               resets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """x, gate, out_gate [B,T,D] (f32 / f16 / bf16, any strides with a contiguous last
    dimension) -> (y [B,T,D], h_last [B,D] float32).

    h0 [B,D] float32 starts the state (zeros without it).  lengths [B]: steps at and
    beyond a row's length leave its state, give y = 0 and are not looked at.  resets
    [B,T] bool: where true the state before that step is dropped (a document starts),
    an infinite or NaN one as well.  Differentiable in x, gate, out_gate and h0 (reverse
    mode, once).
    """
    y, h = _hsru.gated_scan(x, gate, out_gate, h0, lengths, resets)
    return y, h


def gated_scan_packed(packed: torch.Tensor, h0: Optional[torch.Tensor] = None,
                      lengths: Optional[torch.Tensor] = None, resets: Optional[torch.Tensor] = None,
                      out_gate: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """gated_scan of one projection's output [B,T,3D], the concatenation of x, gate and
    out_gate ([B,T,2D] with out_gate=False).  The gradient is one packed tensor too, so
    neither direction copies the parts together."""
    y, h = _hsru.gated_scan_packed(packed, h0, lengths, resets, out_gate)
    return y, h


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, h: torch.Tensor,
                    out_gate: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token: x, gate, out_gate [B,D], h [B,D] float32 updated in place -> y [B,D].
    No backward pass; h counts as changed for one that has saved it."""
    return _hsru.gated_scan_step(x, gate, h, out_gate)


class GatedRecurrence(nn.Module):
    """x [b,t,d] -> out_proj(gated_scan(proj(x))), with DeltaGridLayer's forward / step
    shape: each returns (output, state), the state [b,d] float32."""

    def __init__(self, d_model: int, gate_init: float = 3.0):
        super().__init__()
        self.d_model = d_model
        self.proj = nn.Linear(d_model, 3 * d_model, bias=True)
        self.out_proj = nn.Linear(d_model, d_model, bias=False)
        with torch.no_grad():
            self.proj.bias.zero_()
            self.proj.bias[d_model:2 * d_model].fill_(gate_init)      # memories of about e^gate_init steps

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None,
                resets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        y, state = gated_scan_packed(self.proj(x), state, lengths, resets)
        return self.out_proj(y), state

    def step(self, x: torch.Tensor, state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One token x [b,1,d]; the state is updated in place."""
        b, t, d = x.shape
        if t != 1:
            raise ValueError(f"step() expects sequence length 1, got {t}")
        if state is None:
            state = torch.zeros(b, d, device=x.device, dtype=torch.float32)
        p = self.proj(x.squeeze(1))
        y = gated_scan_step(p[:, :d], p[:, d:2 * d], state, p[:, 2 * d:])
        return self.out_proj(y).unsqueeze(1), state


__all__ = ["gated_scan", "gated_scan_packed", "gated_scan_step", "GatedRecurrence"]
