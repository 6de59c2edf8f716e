"""Gradients of a linear attention without heads: q and k reach no output."""
import pytest
import torch

from mamba_amd.ops.linear_attn import linear_attn_fn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("decays", ["token", "head"])
def test_no_heads(decays):
    q, k = (torch.randn(2, 50, 3, 16, device=DEV).requires_grad_() for _ in range(2))
    v = torch.zeros(2, 50, 0, 16, device=DEV).requires_grad_()
    g = torch.zeros((2, 50, 0) if decays == "token" else (0,), device=DEV).requires_grad_()
    dirty = [torch.full((2, 50, 3, 16), 7.0, device=DEV) for _ in range(4)]       # what the allocator hands out next
    torch.cuda.synchronize()
    del dirty
    out = linear_attn_fn(q, k, v, g)
    dq, dk, dv, dg = torch.autograd.grad(out.sum(), [q, k, v, g])
    assert out.shape == v.shape and dv.shape == v.shape and dg.shape == g.shape
    assert not dq.any() and not dk.any()
