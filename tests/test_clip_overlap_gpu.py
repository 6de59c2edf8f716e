"""clip_grads refuses outputs that lie over other tensors, and takes what only looks like it."""
import pytest
import torch

from mamba_amd.ops.clip_grads import clip_grads

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_overlapping_gradients():
    flat = torch.randn(1000, device=DEV)
    before = flat.clone()
    g = flat[:300].view(10, 30)
    for grads, out in (([g, g], None), ([g, flat[299:400]], None), ([g, flat[500:600]], [flat[400:700].view(10, 30), flat[600:700]]),
                       ([g], [flat[1:301].view(10, 30)]), ([g, flat[500:600]], [torch.empty_like(g), flat[:100]])):
        with pytest.raises(ValueError, match="lies over another tensor"):
            clip_grads(grads, 1.0, out=out)
    assert torch.equal(flat, before)
    # neighbours, empty tensors inside others, and one gradient read twice into outputs apart
    norm = clip_grads([g, flat[300:400], flat[50:50]], 1e9)
    assert abs(float(norm) - float(before[:400].norm())) <= 1e-5 * float(norm) and torch.equal(flat, before)
    out = [torch.empty_like(g), torch.empty_like(g)]
    clip_grads([g, g], 1e9, out=out)
    assert torch.equal(out[0], g) and torch.equal(out[1], g)
