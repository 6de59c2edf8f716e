"""The norm over all gradients of a model, and the gradients clipped to it, on the HIP library.

``clip_grads(grads, max_norm, out=None, eps=1e-6)``: grads is an iterable of
GPU tensors (fp32, bf16 or fp16, of any sizes and mixed dtypes; None entries,
parameters without a gradient, are left out):

    norm = sqrt(sum of all elements' squares)       (64-bit sums)
    out  = grad * min(1, max_norm / (norm + eps))   (fp32, rounded to the tensor's dtype)

The gradients are scaled in place, or written to ``out``, tensors of the same
shapes, strides and dtypes (None where grads holds None).  An output that lies
over another tensor than its own gradient (one gradient given twice, in place) is
refused.  Returns norm, a 0-d
fp32 tensor on the device: nothing waits for the GPU.  Sums have a fixed
order, the same bits on every run.  An infinity or NaN among the gradients
makes the norm infinite or NaN, and the gradients zero (and NaN at the
infinities) or NaN: a training loop looks at the norm and leaves the step out.
"""
import torch

from .. import _native as nat
from ..selective_scan import _raw_stream


def clip_grads(grads, max_norm, out=None, eps=1e-6):
    """Clips gradients by their global norm; see the module docstring."""
    grads = list(grads)
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"clip_grads: out holds {len(outs)} tensors, expected {len(grads)}")
    gs = [g for g in grads if g is not None]
    os = gs if out is None else [o for g, o in zip(grads, outs) if g is not None]
    dev = gs[0].device if gs else torch.device("cuda", torch.cuda.current_device())
    return nat.host().clip_grads(gs, os, float(max_norm), float(eps), dev.index or 0, _raw_stream(dev))
