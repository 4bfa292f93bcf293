"""Gated feed-forward block: both projections, the activation and the product in one
kernel, with its backward pass.

    h = act(x Wg^T + bg) * (x Wu^T + bu)

``weight`` [2F, D] holds the F gate rows, then the F value rows (one nn.Linear's weight).
dg_gated_ffn_forward / _backward in include/deltagrid_b200.h hold the exact contract.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _hsru

_ACT = {"silu": 0, "gelu": 1}


def gated_ffn(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
              activation: str = "silu") -> torch.Tensor:
    """x [..., D], weight [2F, D], bias [2F] (one dtype: f32 / f16 / bf16) -> h [..., F].

    activation "silu" or "gelu" (the tanh form).  Differentiable in x, weight and bias; the
    backward pass forms both projections again, so nothing of size [..., 2F] is kept.  The
    gradients of the projections are rounded to the tensors' type once, before the products
    that use them (f16: its range).  Under torch.autocast it runs in autocast's type, as
    nn.Linear does.
    """
    code = _ACT.get(activation)
    if code is None:
        raise ValueError(f"gated_ffn: activation must be one of {sorted(_ACT)}, got {activation!r}")
    return _hsru.gated_ffn(x, weight, bias, code)


class GatedFFN(nn.Module):
    """fc2(act(gate) * value) with gate and value the halves of fc1."""

    def __init__(self, d_model: int, d_hidden: Optional[int] = None, bias: bool = True, activation: str = "silu"):
        super().__init__()
        d_hidden = d_model if d_hidden is None else d_hidden
        self.activation = activation
        self.fc1 = nn.Linear(d_model, 2 * d_hidden, bias=bias)
        self.fc2 = nn.Linear(d_hidden, d_model, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.fc2(gated_ffn(x, self.fc1.weight, self.fc1.bias, self.activation))


__all__ = ["gated_ffn", "GatedFFN"]
