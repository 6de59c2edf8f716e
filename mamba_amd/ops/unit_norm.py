"""Rows scaled to length one, on the HIP library: the queries and keys of the delta rule.

    out = x * rsqrt(sum(x**2, -1) + eps)

``unit_norm_fn(x, eps=1e-6)``: x of any shape and of fp32, bf16 or fp16, normalised
over its last dim (of up to 16384) in fp32 and rounded once.  The heads of a
projection's output (a slice viewed as (..., heads, dim)) are read where they
lie, queries and keys beside each other in one call.  Gradients flow to x.
Forward-mode and second derivatives are refused.
"""
from .. import _native as nat


def unit_norm_fn(x, eps=1e-6):
    """x scaled to length one along its last dim; see the module docstring."""
    return nat.host().unit_norm(x, float(eps))
