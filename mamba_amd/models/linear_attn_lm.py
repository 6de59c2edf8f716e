"""LinearAttnLM: a language model of LinearAttn mixers with a norm on both sides of each block.

Block i computes y = mixer_i(normed); the border to the next one is a single
call, block_norm_fn: the norm after the block, its residual scale, and the
norm in front of block i + 1 (after the last block: in front of the head).

    normed, s = rms_norm_fn(embedding, pre_0), embedding
    y         = mixer_i(normed)
    normed, s = block_norm_fn(y, s, post_i, pre_{i+1}, scale=scale_i)
    logits    = lm_head(normed)
"""
from dataclasses import dataclass

import torch
import torch.nn as nn

from ..modules.linear_attn import LinearAttn
from ..ops.block_norm import block_norm_fn
from ..ops.rms_norm import rms_norm_fn


@dataclass
class LinearAttnLMConfig:
    vocab_size: int = 32000
    model_dim: int = 512
    num_layers: int = 5
    head_dim: int = 64
    n_groups: int = None
    expansion_factor: int = 2
    residual_scale: float = 0.5
    eps: float = 1e-6


class LinearAttnLM(nn.Module):
    def __init__(self, config: LinearAttnLMConfig, device=None, dtype=None):
        super().__init__()
        self.config = config
        fk = {"device": device, "dtype": dtype}
        d, n = config.model_dim, config.num_layers
        self.embedding = nn.Embedding(config.vocab_size, d, **fk)
        self.mixers = nn.ModuleList([LinearAttn(d, config.head_dim, n_groups=config.n_groups, eps=config.eps,
                                                expansion_factor=config.expansion_factor, **fk) for _ in range(n)])
        self.pre = nn.ParameterList([nn.Parameter(torch.zeros(d, **fk)) for _ in range(n + 1)])
        self.post = nn.ParameterList([nn.Parameter(torch.zeros(d, **fk)) for _ in range(n)])
        self.scale = nn.ParameterList([nn.Parameter(torch.full((d,), config.residual_scale, **fk)) for _ in range(n)])
        self.lm_head = nn.Linear(d, config.vocab_size, bias=False, **fk)

    def _blocks(self, s, mix):
        """mix(i, normed) -> block i's output; returns the head's input."""
        normed = rms_norm_fn(s, self.pre[0], eps=self.config.eps)
        for i in range(len(self.mixers)):
            # (under autocast the mixer's output has 16 bits; the residual stream keeps its type)
            y = mix(i, normed).to(s.dtype)
            normed, s = block_norm_fn(y, s, self.post[i], self.pre[i + 1], scale=self.scale[i], eps=self.config.eps)
        return normed

    def forward(self, input_ids, lengths=None, states=None):
        """Logits (batch, seqlen, vocab).  ``states`` (from allocate_states) are read as what came
        before and left holding the state after each row's last token."""
        def mix(i, normed):
            if states is None:
                return self.mixers[i](normed, lengths=lengths)
            y, states[i] = self.mixers[i](normed, state=states[i], lengths=lengths, return_state=True)
            return y
        return self.lm_head(self._blocks(self.embedding(input_ids), mix))

    def allocate_states(self, batch_size, device=None):
        return [m.allocate_state(batch_size, device) for m in self.mixers]

    @torch.no_grad()
    def step(self, input_ids, states):
        """One token per sequence: input_ids (batch,) -> logits (batch, vocab); the states advance in place.  No gradients flow."""
        return self.lm_head(self._blocks(self.embedding(input_ids), lambda i, normed: self.mixers[i].step(normed, states[i])))

    @torch.no_grad()
    def generate(self, input_ids, max_new_tokens, lengths=None):
        """Greedy continuation, (batch, max_new_tokens); rows of input_ids hold lengths[b] tokens
        (at least one, all of a row's where lengths[b] is larger)."""
        batch, seqlen = input_ids.shape
        if lengths is None:
            at = torch.full((batch,), seqlen, device=input_ids.device)
        else:
            if lengths.shape != (batch,):
                raise ValueError(f"generate: lengths has shape {tuple(lengths.shape)}, expected {(batch,)}")
            at = lengths.long().clamp(max=seqlen)
        if seqlen == 0 or bool((at < 1).any()):
            raise ValueError("generate: a row without a token has nothing to continue")
        if max_new_tokens < 1:
            return input_ids.new_empty(batch, 0)
        states = self.allocate_states(batch, input_ids.device)
        logits = self(input_ids, lengths=lengths, states=states)
        logits = logits[torch.arange(batch, device=input_ids.device), at - 1]
        out = []
        for i in range(max_new_tokens):
            out.append(logits.argmax(-1))
            if i + 1 < max_new_tokens:
                logits = self.step(out[-1], states)
        return torch.stack(out, 1)
