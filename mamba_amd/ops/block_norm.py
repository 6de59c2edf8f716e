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
in a fixed order, so they have the same bits on every run.
"""
import torch

from .. import _native as nat
from ..selective_scan import _raw_stream


class BlockNormFn(torch.autograd.Function):
    """Autograd of block_norm_fn; returns (out, s)."""

    @staticmethod
    def forward(ctx, x, residual, post, pre, gate, scale_vec, scale, eps):
        need = any(ctx.needs_input_grad[:6])
        out, s, rstd, read = nat.host().block_norm_fwd(x, residual, gate, post, pre, scale_vec, scale, eps, need,
                                                       _raw_stream(x.device))
        if need:
            ctx.save_for_backward(*read, rstd)
            ctx.w_dtypes = [None if w is None else w.dtype for w in (post, pre, scale_vec)]
        ctx.scale, ctx.shape = scale, x.shape
        ctx.set_materialize_grads(False)
        return out.view(x.shape), s.view(x.shape)

    @staticmethod
    def backward(ctx, dout, ds):
        if dout is None and ds is None:
            return (None,) * 8
        x, residual, gate, post, pre, scale_vec, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dres, dgate, *dws = nat.host().block_norm_bwd(
            x, residual, gate, post, pre, scale_vec, rstd, ctx.scale, None if dout is None else dout.reshape(x.shape),
            None if ds is None else ds.reshape(x.shape), need[1], _raw_stream(x.device))
        dpost, dpre, dscale = (None if dw is None or not n else dw.to(t) for dw, n, t in
                               zip(dws, (need[2], need[3], need[5]), ctx.w_dtypes))
        return (dx.view(ctx.shape) if need[0] else None, dres.view(ctx.shape) if need[1] else None, dpost, dpre,
                dgate.view(ctx.shape) if gate is not None and need[4] else None, dscale, None, None)


def block_norm_fn(x, residual, post, pre, gate=None, scale=1.0, eps=1e-6):
    """The norm after a block, its gate and residual scale, and the next block's norm; see the module docstring."""
    vec = scale if isinstance(scale, torch.Tensor) else None
    return BlockNormFn.apply(x, residual, post, pre, gate, vec, 1.0 if vec is not None else float(scale), float(eps))


class GatedRMSNormFn(torch.autograd.Function):
    """Autograd of gated_rms_norm_fn."""

    @staticmethod
    def forward(ctx, x, gate, weight, n_groups, eps):
        out, *read = nat.host().gated_norm_fwd(x, gate, weight, n_groups, eps, _raw_stream(x.device))
        if any(ctx.needs_input_grad[:3]):
            ctx.save_for_backward(*read)
        ctx.n_groups, ctx.eps, ctx.shape, ctx.w_dtype = n_groups, eps, x.shape, weight.dtype
        return out.view(x.shape)

    @staticmethod
    def backward(ctx, dout):
        x, gate, weight = ctx.saved_tensors
        dx, dgate, dw = nat.host().gated_norm_bwd(x, gate, weight, dout.reshape(x.shape), ctx.n_groups, ctx.eps,
                                                  _raw_stream(x.device))
        need = ctx.needs_input_grad
        return (dx.view(ctx.shape) if need[0] else None, dgate.view(ctx.shape) if need[1] else None,
                dw.to(ctx.w_dtype) if need[2] else None, None, None)


def gated_rms_norm_fn(x, gate, weight, n_groups=1, eps=1e-6):
    """The gated norm of each of n_groups parts of a row; see the module docstring."""
    return GatedRMSNormFn.apply(x, gate, weight, int(n_groups), float(eps))
