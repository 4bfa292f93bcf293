"""Trains a small HybridLM to repeat a random word that it has seen once, then generates.

    python examples/hybrid_lm.py [--steps 400] [--dtype bf16]

Each sequence is a random word of 8 letters, repeated: after the first copy every letter can
be told from the one 8 places before it.  The loss on the repeated part falls from log(64)
towards 0 and greedy generation continues the word.
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from deltagrid_b200.hybrid import HybridLM  # noqa: E402

VOCAB, WORD, REPEATS = 64, 8, 8


def batch(n: int, generator: torch.Generator) -> torch.Tensor:
    word = torch.stack([torch.randperm(VOCAB, device="cuda", generator=generator)[:WORD] for _ in range(n)])
    return word.repeat(1, REPEATS)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--dtype", choices=["f32", "bf16"], default="f32")
    args = ap.parse_args()
    torch.manual_seed(0)
    gen = torch.Generator(device="cuda").manual_seed(0)
    model = HybridLM(VOCAB, d_model=256, layers=4, num_heads=4).cuda()
    if args.dtype == "bf16":
        model = model.bfloat16()
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    for i in range(args.steps):
        ids = batch(args.batch, gen)
        logits, _ = model(ids[:, :-1])
        loss = F.cross_entropy(logits[:, WORD - 1:].float().reshape(-1, VOCAB), ids[:, WORD:].reshape(-1))
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if i % 50 == 0 or i == args.steps - 1:
            print(f"step {i:4d}  loss {loss.item():.4f}")
    ids = batch(16, gen)
    tokens, logprobs = model.eval().generate(ids[:, :2 * WORD], 2 * WORD, temperature=0.0)
    print("greedy letters right:", (tokens == ids[:, :2 * WORD]).float().mean().item())
    tokens, logprobs = model.generate(ids[:, :2 * WORD], 2 * WORD, temperature=0.8, top_k=8, top_p=0.95,
                                      generator=torch.Generator(device="cuda").manual_seed(1))
    print("drawn letters right: ", (tokens == ids[:, :2 * WORD]).float().mean().item(),
          " mean log-probability", logprobs.mean().item())


if __name__ == "__main__":
    main()
