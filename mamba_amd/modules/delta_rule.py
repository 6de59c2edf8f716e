"""DeltaRule: LinearAttn's relative whose state is corrected towards each value (absent in the reference).

    qk, v, z, dt, b = split(input_proj(h))
    q, k = split(unit_norm_fn(qk))                      each head's rows of length one (ops/unit_norm.py)
    g    = -exp(log_A) * softplus(dt + dt_bias)         log decay of each head and token
    beta = sigmoid(b)                                   its rate
    o    = delta_rule_fn(q, k, v, g, beta)              (ops/delta_rule.py)
    out  = output_proj(gated_rms_norm_fn(o, z, norm))   each head's norm and gate (ops/block_norm.py)

``forward`` runs prompts and training, over rows of different ``lengths`` and
from a ``state`` of earlier tokens; ``step`` advances the state by one token,
without gradients.
All on the HIP library: tensors on a ROCm device.
"""
import torch
import torch.nn.functional as F

from ..ops.block_norm import gated_rms_norm_fn
from ..ops.delta_rule import delta_rule_fn, delta_rule_update
from ..ops.unit_norm import unit_norm_fn
from .linear_attn import LinearAttn


class DeltaRule(LinearAttn):
    def _sizes(self, qk):
        return [2 * qk, self.inner_dim, self.inner_dim, self.n_heads, self.n_heads]

    def _split(self, hidden_states):
        qk, v, z, dt, b = self.input_proj(hidden_states).split(self.sizes, -1)
        g = -torch.exp(self.log_A.float()) * F.softplus(dt.float() + self.dt_bias.float())
        lead = hidden_states.shape[:-1]
        q, k = unit_norm_fn(qk.view(*lead, 2 * self.n_groups, self.key_dim), self.eps).chunk(2, -2)
        return q, k, v.view(*lead, self.n_heads, self.head_dim), z, g, torch.sigmoid(b.float())

    def forward(self, hidden_states, state=None, lengths=None, return_state=False):
        """(batch, seqlen, model_dim) -> the same shape, or (it, the state after each row's last token)."""
        q, k, v, z, g, beta = self._split(hidden_states)
        o, last = delta_rule_fn(q, k, v, g, beta, initial_state=state, lengths=lengths, return_last_state=True)
        out = self.output_proj(gated_rms_norm_fn(o.flatten(2), z, self.norm, n_groups=self.n_heads, eps=self.eps))
        return (out, last) if return_state else out

    @torch.no_grad()
    def step(self, hidden_states, state):
        """One token: (batch, model_dim) -> the same shape; the state advances in place.  No gradients flow."""
        q, k, v, z, g, beta = self._split(hidden_states)
        o = delta_rule_update(state, q, k, v, g, beta)
        return self.output_proj(gated_rms_norm_fn(o.flatten(1), z, self.norm, n_groups=self.n_heads, eps=self.eps))
