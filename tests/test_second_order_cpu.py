"""Gradients that are final: their own derivative is refused, their values stay."""
import pytest
import torch

from mamba_amd import _native as nat


def test_final_gradients():
    t = [torch.randn(3, 4), None, torch.randn(5).half(), torch.zeros(0)]
    got = nat.host().final_grads("op", t)
    assert got[1] is None
    for a, b in ((got[0], t[0]), (got[2], t[2]), (got[3], t[3])):
        assert torch.equal(a.detach(), b) and a.dtype == b.dtype and a.requires_grad and not a._is_view()
    with pytest.raises(RuntimeError, match="op: .*second"):
        (got[0].square().sum() + got[2].float().sum()).backward()
    kept = torch.randn(3, 4, requires_grad=True)
    (kept.square().sum() + got[0].detach().sum()).backward()
    assert torch.equal(kept.grad, 2 * kept.detach())
    with torch.no_grad():
        got[0].mul_(2.0)
