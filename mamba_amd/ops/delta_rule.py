"""The gated delta rule, on the HIP library.

Linear attention whose state is corrected towards each value instead of added to
(the reference has no such operator).  Per head, with the log decay g (at most 0
where the state decays), a = exp(g), and the rate beta (0 to 1, or to 2):

    e_t = v_t - a_t S_{t-1}^T k_t                 what the state gets wrong
    S_t = a_t S_{t-1} + beta_t k_t e_t^T          (d_key x d_value, fp32)
    out_t = scale * S_t^T q_t

Keys of length one (ops/unit_norm.py) keep the state bounded; longer ones than
sqrt(2 / beta) let it grow from token to token, as the formula says.

``delta_rule_fn(q, k, v, g, beta, scale=None, initial_state=None, lengths=None,
return_last_state=False)``: q, k (batch, seqlen, groups, d_key) and v (batch,
seqlen, heads, d_value) share a dtype (fp32, bf16 or fp16); heads is a multiple
of groups, and heads h of one group share q and k (h // (heads // groups)).
d_key and d_value are 1 to 256.  g and beta are (batch, seqlen, heads) in fp32 or
v's dtype, expanded tensors too; a g of minus infinity empties the state before its
token.  scale defaults to d_key ** -0.5.  initial_state: fp32 (batch, heads, d_key,
d_value), the state before the first token (zero when None).  lengths: (batch,)
integers, row b holds its first lengths[b] tokens: what lies past them is not
read and gets zero outputs and gradients, and the row's last state is the one
after its own last token (a row of length 0 keeps its initial state).  Returns
out (batch, seqlen, heads, d_value), or (out, last_state) with
``return_last_state``.  Gradients flow to q, k, v, g, beta and initial_state;
their sums have a fixed order, so the same bits on every run, and every term of
dg has the factor exp(g): it is zero where the decay empties the state.  With
gradients, a state for each 32 or 64 tokens is kept until the backward.
Tokens are computed in chunks of up to 64: a token's infinities or NaN reach the outputs
of its whole chunk, earlier tokens among them, and of later ones.
Forward-mode and second derivatives are refused.

``delta_rule_update(state, q, k, v, g, beta, scale=None, out=None)`` advances
state (batch, heads, d_key, d_value) by one token in place: q, k (batch, groups,
d_key), v (batch, heads, d_value), g, beta (batch, heads); returns out
(batch, heads, d_value).  The state after a prompt is delta_rule_fn's
last_state.  Elements of state or of out that share memory (an expanded state)
are refused; neither may lie over another tensor of the call.  It has no
backward: with grad mode on, inputs that require a gradient are refused.
"""
from .. import _native as nat
from ..selective_scan import _raw_stream


def delta_rule_fn(q, k, v, g, beta, scale=None, initial_state=None, lengths=None, return_last_state=False):
    """The gated delta rule over rows of tokens; see the module docstring."""
    if scale is None:
        scale = max(1, q.shape[-1]) ** -0.5
    out, last = nat.host().delta_rule(q, k, v, g, beta, initial_state, lengths, float(scale), bool(return_last_state))
    return (out, last) if return_last_state else out


def delta_rule_update(state, q, k, v, g, beta, scale=None, out=None):
    """One token of delta_rule_fn from ``state``, which advances in place; see the module docstring."""
    if scale is None:
        scale = max(1, q.shape[-1]) ** -0.5
    return nat.host().delta_update(state, q, k, v, g, beta, float(scale), out, _raw_stream(v.device))
