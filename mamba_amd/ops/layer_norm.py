"""Layer norm (+ residual add) on the HIP library.

The relative of rms_norm_fn that takes the mean off (the reference has RMSNorm only):

    s   = x + residual            (rounded to x's dtype; s = x without residual)
    out = (s - mean(s)) * rsqrt(mean((s - mean(s))**2, -1) + eps) * weight + bias

in fp32, over the last dim, rounded once to x's dtype.

``layer_norm_fn(x, weight, bias=None, residual=None, eps=1e-5, prenorm=False)``
returns out, or (out, s) when ``prenorm`` (s is the residual stream that the next
block adds to; x without residual).  x and residual share shape and dtype
(fp32, bf16 or fp16; rows of up to 16384); weight and bias are (dim,) of any float
dtype (read as fp32 unless all are of x's dtype).  Gradients flow to x, weight, bias
and residual; weight and bias gradients are summed over rows in a fixed order, so
they have the same bits on every run.  Forward-mode and second derivatives are refused.
"""
from .. import _native as nat


def layer_norm_fn(x, weight, bias=None, residual=None, eps=1e-5, prenorm=False):
    """Layer norm of x (+ residual) on the HIP kernels; see the module docstring."""
    out, s = nat.host().layer_norm(x, weight, bias, residual, float(eps), bool(prenorm))
    if not prenorm:
        return out
    return out, x if s is None else s
