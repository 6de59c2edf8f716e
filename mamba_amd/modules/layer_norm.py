"""LayerNorm: RMSNorm's relative that takes the mean off, with the same residual and prenorm (absent in the reference).

out = (s - mean(s)) * rsqrt(var(s) + eps) * weight + bias, computed in fp32 and cast
back to x's dtype; weight starts at one, bias (left out with ``bias=False``) at zero.

``forward(x, residual=None, prenorm=False)`` normalises s = x + residual (rounded to x's dtype),
and with ``prenorm`` returns (out, s).  On a ROCm device this is one HIP kernel
(``mamba_amd.ops.layer_norm``); elsewhere PyTorch ops.
"""
import torch
import torch.nn as nn

from ..ops.layer_norm import layer_norm_fn


class LayerNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if bias else None

    def forward(self, x, residual=None, prenorm=False):
        if x.is_cuda:
            return layer_norm_fn(x, self.weight, self.bias, residual, self.eps, prenorm)
        if residual is not None:
            x = x + residual
        xf = x.float()
        c = xf - xf.mean(-1, keepdim=True)
        out = c * torch.rsqrt(c.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight.float()
        if self.bias is not None:
            out = out + self.bias.float()
        out = out.type_as(x)
        return (out, x) if prenorm else out
