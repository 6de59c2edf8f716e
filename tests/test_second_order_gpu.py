"""The scan, the block, the conv and RMSNorm refuse a derivative of their gradients
where plain tensors would drop it; gradients kept with a graph are as without."""
import pytest
import torch

from mamba_amd.modules.mamba_simple import MambaSimple
from mamba_amd.ops.causal_conv1d import causal_conv1d_fn
from mamba_amd.ops.rms_norm import rms_norm_fn
from mamba_amd.ops.selective_scan_interface import SelectiveScanFn, selective_scan_fn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def calls():
    torch.manual_seed(0)

    def r(*s):
        return torch.randn(s, device=DEV)

    block = MambaSimple(32, device=DEV)
    scan = [r(1, 16, 40), r(1, 16, 40) * 0.1, -r(16, 16).exp(), r(1, 1, 16, 40), r(1, 1, 16, 40), r(16)]
    return {
        "scan": (SelectiveScanFn.apply, scan),
        "scan-z": (lambda u, dt, A, B, C, D, z: selective_scan_fn(u, dt, A, B, C, D, z=z, delta_softplus=True), scan + [r(1, 16, 40)]),
        "block": (block, [r(1, 20, 32)]),
        "conv": (lambda x, w, b: causal_conv1d_fn(x, w, b, "silu"), [r(1, 16, 40), r(16, 4), r(16)]),
        "rms_norm": (lambda x, w, s: rms_norm_fn(x, w, s), [r(5, 24), r(24), r(5, 24)]),
        "rms_norm prenorm": (lambda x, w, s: sum(rms_norm_fn(x, w, s, prenorm=True)), [r(5, 24), r(24), r(5, 24)]),
    }


@pytest.mark.parametrize("name", ["scan", "scan-z", "block", "conv", "rms_norm", "rms_norm prenorm"])
def test_second_derivatives_are_refused(name):
    call, x = calls()[name]
    for n in range(len(x)):
        y = [t.clone() for t in x]
        y[n].requires_grad_()
        first, = torch.autograd.grad(call(*y).sum(), [y[n]])
        graph, = torch.autograd.grad(call(*y).sum(), [y[n]], create_graph=True)
        # (dB and dC are sums by atomics: their order, and what follows from them, changes between runs)
        assert (first - graph.detach()).abs().max() <= 2.0 ** -14 * first.abs().max()
        with pytest.raises(RuntimeError, match="second"):
            (graph.square().sum() + y[n].square().sum()).backward()
