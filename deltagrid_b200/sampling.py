"""Token sampling with temperature, top-k, top-p and min-p from given uniform numbers.

The masses exp((l - max) / temperature) are 40-bit fixed-point integers and their sums
64-bit, so a row's token depends on its logits, parameters and number alone: not on the
batch it is in, the order of a reduction or the device's load.  dg_sample in
include/deltagrid_b200.h holds the exact contract.
"""
from __future__ import annotations

from typing import Tuple, Union

import torch

from . import _hsru

Number = Union[int, float, torch.Tensor]


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Number = 1.0, top_k: Number = 0,
           top_p: Number = 1.0, min_p: Number = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """logits [B,V] (f32 / f16 / bf16, any row stride), u [B] float32 in [0, 1) ->
    (token [B] int64, logprob [B] float32 under the filtered distribution).

    Each parameter is a number or a [B] tensor.  temperature <= 0 takes the largest logit
    (lowest index); top_k <= 0 keeps all.  NaN logits count as -inf; a row of -inf gives
    token -1 and logprob -inf.  V is 2^18 at most.  Not differentiable: logprob carries no
    gradient.
    """
    t, tv = (temperature, 0.0) if isinstance(temperature, torch.Tensor) else (None, temperature)
    k, kv = (top_k, 0) if isinstance(top_k, torch.Tensor) else (None, top_k)
    p, pv = (top_p, 0.0) if isinstance(top_p, torch.Tensor) else (None, top_p)
    m, mv = (min_p, 0.0) if isinstance(min_p, torch.Tensor) else (None, min_p)
    token, logprob = _hsru.sample(logits, u, t, tv, k, kv, p, pv, m, mv)
    return token, logprob


__all__ = ["sample"]
