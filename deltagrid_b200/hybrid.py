"""A small hybrid recurrent language model on this package's kernels, trained and served.

Blocks alternate two mixers, the gated linear recurrence (cheap, fading memory of a fixed
size) and DeltaGridLayer (associative memory), each followed by the gated feed-forward block:

    x = x + mixer(norm(x));    x = x + ffn(norm(x))

``forward`` runs sequences (training, prefill), ``step`` one token per sequence on the
states that ``forward`` returns, and ``generate`` draws tokens with sampling.sample.  All
state has a fixed size: there is no cache that grows with the sequence.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
import torch.nn as nn

from .ffn import GatedFFN
from .layer import DeltaGridLayer
from .recurrence import GatedRecurrence
from .sampling import sample


class HybridBlock(nn.Module):
    """kind "recurrence" or "delta"; forward and step return (x, state).  resets (where documents start) are
    for the recurrence: the memory layer's state cannot be dropped inside a sequence."""

    def __init__(self, kind: str, d_model: int, num_heads: int, num_slots: Optional[int], d_hidden: Optional[int],
                 activation: str = "silu"):
        super().__init__()
        if kind not in ("recurrence", "delta"):
            raise ValueError(f"HybridBlock: kind must be 'recurrence' or 'delta', got {kind!r}")
        self.kind = kind
        self.norm_mixer = nn.LayerNorm(d_model)
        self.mixer = (GatedRecurrence(d_model) if kind == "recurrence"
                      else DeltaGridLayer(d_model, num_heads=num_heads, num_slots=num_slots))
        self.norm_ffn = nn.LayerNorm(d_model)
        self.ffn = GatedFFN(d_model, d_hidden, activation=activation)

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                resets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        if resets is not None and self.kind == "delta":
            raise ValueError("HybridBlock: resets are not supported by 'delta' blocks")
        h = self.norm_mixer(x)
        y, state = self.mixer(h, state, resets=resets) if self.kind == "recurrence" else self.mixer(h, state)
        x = x + y
        return x + self.ffn(self.norm_ffn(x)), state

    def step(self, x: torch.Tensor, state: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
        y, state = self.mixer.step(self.norm_mixer(x), state)
        x = x + y
        return x + self.ffn(self.norm_ffn(x)), state


class HybridLM(nn.Module):
    """Token ids -> logits.  ``layers`` blocks, "recurrence" and "delta" in turn."""

    def __init__(self, vocab_size: int, d_model: int = 256, layers: int = 4, num_heads: int = 4,
                 num_slots: Optional[int] = None, d_hidden: Optional[int] = None, activation: str = "silu"):
        super().__init__()
        self.embed = nn.Embedding(vocab_size, d_model)
        self.blocks = nn.ModuleList([HybridBlock("delta" if i % 2 else "recurrence", d_model, num_heads, num_slots,
                                                 d_hidden, activation) for i in range(layers)])
        self.norm = nn.LayerNorm(d_model)
        self.head = nn.Linear(d_model, vocab_size, bias=False)

    def forward(self, ids: torch.Tensor, states: Optional[List[torch.Tensor]] = None
                ) -> Tuple[torch.Tensor, List[torch.Tensor]]:
        """ids [B,T] -> (logits [B,T,V], one state per block)."""
        x = self.embed(ids)
        out = []
        for i, block in enumerate(self.blocks):
            x, s = block(x, states[i] if states is not None else None)
            out.append(s)
        return self.head(self.norm(x)), out

    def step(self, ids: torch.Tensor, states: List[torch.Tensor]) -> Tuple[torch.Tensor, List[torch.Tensor]]:
        """ids [B], the last token of each sequence -> (logits [B,V], states); the recurrence's
        states are updated in place."""
        x = self.embed(ids).unsqueeze(1)
        out = []
        for block, s in zip(self.blocks, states):
            x, s = block.step(x, s)
            out.append(s)
        return self.head(self.norm(x)).squeeze(1), out

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, max_new_tokens: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 u: Optional[torch.Tensor] = None, generator: Optional[torch.Generator] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
        """Continues the prompts ids [B,T] (T >= 1) -> (new tokens [B,N], their log-probabilities
        [B,N] under the filtered distributions).

        u [B,N] float32 in [0, 1): the uniform numbers to draw with; without it they are taken
        from ``generator``.  The other arguments are sampling.sample's.  Where nothing can be drawn (all
        of a row's logits NaN or -inf) the token is -1, its log-probability -inf, and the row goes on
        from token 0.
        """
        if ids.dim() != 2 or ids.shape[1] == 0:
            raise ValueError(f"generate: expected prompts [B,T] with at least one token, got {tuple(ids.shape)}")
        B = ids.shape[0]
        if u is None:
            u = torch.rand(B, max_new_tokens, device=ids.device, generator=generator)
        elif tuple(u.shape) != (B, max_new_tokens):
            raise ValueError(f"generate: expected u [{B},{max_new_tokens}], got {tuple(u.shape)}")
        tokens = torch.empty(B, max_new_tokens, dtype=torch.int64, device=ids.device)
        logprobs = torch.empty(B, max_new_tokens, dtype=torch.float32, device=ids.device)
        if max_new_tokens == 0:
            return tokens, logprobs
        logits, states = self(ids)
        logits = logits[:, -1]
        for i in range(max_new_tokens):
            tokens[:, i], logprobs[:, i] = sample(logits, u[:, i], temperature, top_k, top_p, min_p)
            if i + 1 < max_new_tokens:
                logits, states = self.step(tokens[:, i].clamp(min=0), states)      # (-1 is no row of the embedding)
        return tokens, logprobs


__all__ = ["HybridBlock", "HybridLM"]
