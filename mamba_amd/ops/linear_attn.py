"""Linear attention with a decay for each head, on the HIP library.

The matrix-state relative of the selective scan (the reference has no such
operator).  Per head, with the log decay g (at most 0 where the state decays):

    S_t = exp(g_t) S_{t-1} + k_t v_t^T          (d_key x d_value, fp32)
    out_t = scale * q_t^T S_t

``linear_attn_fn(q, k, v, g, scale=None, initial_state=None, lengths=None,
return_last_state=False)``: q, k (batch, seqlen, groups, d_key) and v (batch,
seqlen, heads, d_value) share a dtype (fp32, bf16 or fp16); heads is a multiple
of groups, and heads h of one group share q and k (h // (heads // groups)).
d_key and d_value are 1 to 256.  g is (batch, seqlen, heads), or (heads,) for
one decay per head, in fp32 or v's dtype; minus infinity empties the state
before its token.  scale defaults to d_key ** -0.5.  initial_state: fp32
(batch, heads, d_key, d_value), the state before the first token (zero when
None).  lengths: (batch,) integers, row b holds its first lengths[b] tokens:
what lies past them is not read and gets zero outputs and gradients, and the
row's last state is the one after its own last token (a row of length 0 keeps
its initial state).  Returns out (batch, seqlen, heads, d_value), or (out,
last_state) with ``return_last_state``.  Gradients flow to q, k, v, g and
initial_state; their sums have a fixed order, so the same bits on every run.
dg of a token is zero where exp(g) is, and within a small part of exp(g) |S| |dS|
(the states on its two sides) where g is below -8.3; above, it is a difference of
sums over up to 1024 tokens, and within about 2^-21 of their size.
A token's infinities or NaN reach the outputs of its own and later tokens (and,
of the gradients, dg of earlier tokens too).
Forward-mode and second derivatives are refused.

``linear_attn_update(state, q, k, v, g, scale=None, out=None)`` advances state
(batch, heads, d_key, d_value) by one token in place: q, k (batch, groups,
d_key), v (batch, heads, d_value), g (batch, heads) or (heads,); returns out
(batch, heads, d_value).  The state after a prompt is linear_attn_fn's
last_state.  Elements of state or of out that share memory (an expanded state)
are refused; neither may lie over another tensor of the call.  It has no
backward: with grad mode on, inputs that require a gradient are refused.
"""
from .. import _native as nat
from ..selective_scan import _raw_stream


def linear_attn_fn(q, k, v, g, scale=None, initial_state=None, lengths=None, return_last_state=False):
    """Linear attention with a decay for each head; see the module docstring."""
    if scale is None:
        scale = max(1, q.shape[-1]) ** -0.5
    out, last = nat.host().linear_attn(q, k, v, g, initial_state, lengths, float(scale), bool(return_last_state))
    return (out, last) if return_last_state else out


def linear_attn_update(state, q, k, v, g, scale=None, out=None):
    """One token of linear_attn_fn from ``state``, which advances in place; see the module docstring."""
    if scale is None:
        scale = max(1, q.shape[-1]) ** -0.5
    return nat.host().lin_update(state, q, k, v, g, float(scale), out, _raw_stream(v.device))
