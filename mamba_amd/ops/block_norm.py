"""The norms around a block, and the gated norm of each head, on the HIP library.

The reference's block has one norm, in front (models/causal_lm.py:30-35).
With rms(v) = v * rsqrt(mean(v**2, -1) + eps) in fp32:

``block_norm_fn(x, residual, post, pre, gate=None, scale=1.0, eps=1e-6)`` is the
border between two blocks, in one pass: the norm after a block, its gate and
residual scale, and the norm in front of the next block:

    t   = rms(x) * (1 + post) (* silu(gate))
    s   = residual + scale * t
    out = rms(s) * (1 + pre)

x, residual and gate share shape and dtype (fp32, bf16 or fp16; rows of up to
16384); post and pre are (dim,); scale is a number or a (dim,) tensor.
Weights of another float dtype than x's are read as fp32.  Returns (out, s),
each computed in fp32 and rounded once to x's dtype; s is the residual stream
of the next border.  Gradients flow to x, residual, post, pre, gate and a
tensor scale.

``gated_rms_norm_fn(x, gate, weight, n_groups=1, eps=1e-6)`` normalises each
of n_groups equal parts of a row (the heads of a block) by itself:

    out = rms(part of x) * (1 + weight) * silu(gate)

Gradients flow to x, gate and weight.  Weight gradients are summed over rows
in a fixed order, so they have the same bits on every run.  Forward-mode and
second derivatives are refused.
"""
import torch

from .. import _native as nat


def block_norm_fn(x, residual, post, pre, gate=None, scale=1.0, eps=1e-6):
    """The norm after a block, its gate and residual scale, and the next block's norm; see the module docstring."""
    vec = scale if isinstance(scale, torch.Tensor) else None
    return nat.host().block_norm(x, residual, post, pre, gate, vec, 1.0 if vec is not None else float(scale), float(eps))


def gated_rms_norm_fn(x, gate, weight, n_groups=1, eps=1e-6):
    """The gated norm of each of n_groups parts of a row; see the module docstring."""
    return nat.host().gated_norm(x, gate, weight, int(n_groups), float(eps))
