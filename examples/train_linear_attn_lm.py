"""Trains a small LinearAttnLM to repeat what it read, and lets it answer.

A sequence is random symbols, a separator and the symbols again; the loss
counts the second half.  Every step runs the chunked linear attention, the
gated norms of the heads, the border norms and the clipping of the gradients
by their global norm; the answers come from prompts of different lengths and
then one token at a time.

    python examples/train_linear_attn_lm.py [--steps 300] [--symbols 8] [--length 12]
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mamba_amd.models.linear_attn_lm import LinearAttnLM, LinearAttnLMConfig  # noqa: E402
from mamba_amd.ops.clip_grads import clip_grads  # noqa: E402


def batch_of(n, symbols, length, gen, device):
    x = torch.randint(1, symbols + 1, (n, length), generator=gen, device=device)
    return torch.cat([x, torch.zeros(n, 1, dtype=x.dtype, device=device), x], 1)


def train(steps=300, symbols=8, length=12, batch=64, lr=3e-3, max_norm=1.0, seed=0, log=print, device="cuda"):
    """Returns (model, losses)."""
    torch.manual_seed(seed)
    gen = torch.Generator(device=device).manual_seed(seed)
    model = LinearAttnLM(LinearAttnLMConfig(vocab_size=symbols + 1, model_dim=64, num_layers=2, head_dim=32), device=device)
    params = list(model.parameters())
    opt = torch.optim.AdamW(params, lr=lr)
    losses = []
    for step in range(steps):
        seq = batch_of(batch, symbols, length, gen, device)
        logits = model(seq[:, :-1])[:, length:]
        loss = F.cross_entropy(logits.reshape(-1, symbols + 1), seq[:, length + 1:].reshape(-1))
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norm = clip_grads([p.grad for p in params], max_norm)
        opt.step()
        losses.append(loss.detach())
        if step % 50 == 0 or step + 1 == steps:
            log(f"step {step:4d}  loss {loss.item():.4f}  gradient norm {norm.item():.3f}")
    return model, [x.item() for x in losses]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--symbols", type=int, default=8)
    ap.add_argument("--length", type=int, default=12)
    a = ap.parse_args()
    model, _ = train(a.steps, a.symbols, a.length)
    gen = torch.Generator(device="cuda").manual_seed(1)
    # prompts of different lengths in one batch: symbols and the separator
    full = batch_of(4, a.symbols, a.length, gen, "cuda")
    n = torch.tensor([max(1, a.length - i) for i in range(4)], device="cuda")
    prompt = torch.zeros(4, a.length + 1, dtype=full.dtype, device="cuda")
    for i in range(4):
        prompt[i, :n[i]] = full[i, :n[i]]
    answers = model.generate(prompt, a.length, lengths=n + 1)
    for i in range(4):
        want, got = full[i, :n[i]].tolist(), answers[i, :n[i]].tolist()
        print(f"read {want}\nsaid {got}  ({sum(x == y for x, y in zip(want, got))} of {len(want)} right)")


if __name__ == "__main__":
    main()
