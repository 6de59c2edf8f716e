"""In-place operations on what the norms return, with and without autograd."""
import pytest
import torch

from mamba_amd.ops.block_norm import block_norm_fn, gated_rms_norm_fn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("grad", [False, True], ids=["plain", "autograd"])
@pytest.mark.parametrize("shape", [(6, 24), (2, 3, 24), (24,)], ids=lambda s: "x".join(map(str, s)))
def test_results_can_be_changed_in_place(shape, grad):
    torch.manual_seed(0)
    x, res, z = (torch.randn(shape, device=DEV).requires_grad_(grad) for _ in range(3))
    w = torch.randn(24, device=DEV)
    out, s = block_norm_fn(x, res, w, w, gate=z)
    h = gated_rms_norm_fn(x, z, w, 3)
    held = [t.detach().clone() for t in (out, s, h)]
    for t, before in zip((out, s, h), held):
        assert t.shape == x.shape and t.is_contiguous()
        t.mul_(2.0)
        assert torch.equal(t.detach(), 2.0 * before)
    if grad:
        got = torch.autograd.grad([out, s, h], [x, res, z], [torch.ones_like(x)] * 3)
        out, s = block_norm_fn(x, res, w, w, gate=z)
        want = torch.autograd.grad([out, s, gated_rms_norm_fn(x, z, w, 3)], [x, res, z], [torch.full_like(x, 2.0)] * 3)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
