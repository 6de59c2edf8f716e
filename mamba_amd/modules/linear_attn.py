"""LinearAttn: a mixer like MambaSimple with a matrix state per head (absent in the reference).

    q, k, v, z, dt = split(input_proj(h))
    g   = -exp(log_A) * softplus(dt + dt_bias)          log decay of each head and token
    o   = linear_attn_fn(q, k, v, g)                    (ops/linear_attn.py)
    out = output_proj(gated_rms_norm_fn(o, z, norm))    each head's norm and gate (ops/block_norm.py)

``forward`` runs prompts and training, over rows of different ``lengths`` and
from a ``state`` of earlier tokens; ``step`` advances the state by one token,
without gradients.
All on the HIP library: tensors on a ROCm device.
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.block_norm import gated_rms_norm_fn
from ..ops.linear_attn import linear_attn_fn, linear_attn_update


class LinearAttn(nn.Module):
    def __init__(self, model_dim, head_dim=64, key_dim=None, n_groups=None, expansion_factor=2, delta_min=0.001,
                 delta_max=0.1, eps=1e-6, device=None, dtype=None):
        super().__init__()
        fk = {"device": device, "dtype": dtype}
        self.inner_dim = int(expansion_factor * model_dim)
        if self.inner_dim % head_dim:
            raise ValueError(f"LinearAttn: {self.inner_dim} channels are no whole number of {head_dim}-wide heads")
        self.n_heads, self.head_dim = self.inner_dim // head_dim, head_dim
        self.key_dim, self.n_groups = key_dim or head_dim, n_groups or self.n_heads
        self.eps = eps
        qk = self.n_groups * self.key_dim
        self.sizes = [qk, qk, self.inner_dim, self.inner_dim, self.n_heads]
        self.input_proj = nn.Linear(model_dim, sum(self.sizes), bias=False, **fk)
        self.norm = nn.Parameter(torch.zeros(self.inner_dim, **fk))
        self.output_proj = nn.Linear(self.inner_dim, model_dim, bias=False, **fk)
        delta = torch.exp(torch.rand(self.n_heads, device=device) * math.log(delta_max / delta_min) + math.log(delta_min))
        self.dt_bias = nn.Parameter(delta + torch.log(-torch.expm1(-delta)))            # softplus of it is delta
        self.log_A = nn.Parameter(torch.log(1 + 15 * torch.rand(self.n_heads, device=device)))

    def _split(self, hidden_states):
        q, k, v, z, dt = self.input_proj(hidden_states).split(self.sizes, -1)
        g = -torch.exp(self.log_A.float()) * F.softplus(dt.float() + self.dt_bias.float())
        lead = hidden_states.shape[:-1]
        qk = (*lead, self.n_groups, self.key_dim)
        return q.reshape(qk), k.reshape(qk), v.reshape(*lead, self.n_heads, self.head_dim), z, g

    def forward(self, hidden_states, state=None, lengths=None, return_state=False):
        """(batch, seqlen, model_dim) -> the same shape, or (it, the state after each row's last token)."""
        q, k, v, z, g = self._split(hidden_states)
        o, last = linear_attn_fn(q, k, v, g, initial_state=state, lengths=lengths, return_last_state=True)
        out = self.output_proj(gated_rms_norm_fn(o.flatten(2), z, self.norm, n_groups=self.n_heads, eps=self.eps))
        return (out, last) if return_state else out

    def allocate_state(self, batch_size, device=None):
        """The state before a sequence starts: fp32 (batch, heads, key_dim, head_dim), zero."""
        device = self.input_proj.weight.device if device is None else device
        return torch.zeros(batch_size, self.n_heads, self.key_dim, self.head_dim, device=device)

    @torch.no_grad()
    def step(self, hidden_states, state):
        """One token: (batch, model_dim) -> the same shape; the state advances in place.  No gradients flow."""
        q, k, v, z, g = self._split(hidden_states)
        o = linear_attn_update(state, q, k, v, g)
        return self.output_proj(gated_rms_norm_fn(o.flatten(1), z, self.norm, n_groups=self.n_heads, eps=self.eps))
