"""Derivatives that the operators do not have are refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from mamba_amd.ops.block_norm import block_norm_fn, gated_rms_norm_fn
from mamba_amd.ops.clip_grads import clip_grads
from mamba_amd.ops.linear_attn import linear_attn_fn, linear_attn_update

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def calls():
    """name -> (call of its tensors, tensors)"""
    torch.manual_seed(0)

    def r(*s):
        return torch.randn(s, device=DEV)

    return {
        "linear_attn": (lambda q, k, v, g, i: linear_attn_fn(q, k, v, g, initial_state=i),
                        [r(1, 40, 2, 16), r(1, 40, 2, 16), r(1, 40, 2, 8), -r(1, 40, 2).abs(), r(1, 2, 16, 8)]),
        "border": (lambda x, res, post, pre, z, sc: block_norm_fn(x, res, post, pre, gate=z, scale=sc)[0],
                   [r(5, 24), r(5, 24), r(24), r(24), r(5, 24), r(24)]),
        "heads": (lambda x, z, w: gated_rms_norm_fn(x, z, w, 3), [r(5, 24), r(5, 24), r(24)]),
    }


FORWARD = ([(n, i) for n, k in (("linear_attn", 5), ("border", 6), ("heads", 3)) for i in range(k)])


@pytest.mark.parametrize("name,which", FORWARD, ids=[f"{n}-{i}" for n, i in FORWARD])
def test_tangents_are_refused(name, which):
    call, x = calls()[name]
    want = call(*x)
    with fwad.dual_level():
        y = list(x)
        y[which] = fwad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(ValueError, match="forward-mode"):
            call(*y)
        assert torch.equal(call(*x), want)


def test_tangents_are_refused_in_place():
    torch.manual_seed(0)
    state, t = torch.randn(1, 2, 16, 8, device=DEV), torch.randn(1, 2, 16, device=DEV)
    v, g = torch.randn(1, 2, 8, device=DEV), torch.zeros(1, 2, device=DEV)
    with fwad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            linear_attn_update(state, fwad.make_dual(t, t), t, v, g)
        with pytest.raises(ValueError, match="forward-mode"):
            clip_grads([fwad.make_dual(t, t)], 1.0)


@pytest.mark.parametrize("name", ["linear_attn", "border", "heads"])
def test_second_derivatives_are_refused(name):
    call, x = calls()[name]
    for n in range(len(x)):
        y = [t.clone() for t in x]
        y[n].requires_grad_()
        first, = torch.autograd.grad(call(*y).sum(), [y[n]])
        graph, = torch.autograd.grad(call(*y).sum(), [y[n]], create_graph=True)
        assert torch.equal(first, graph)
        with pytest.raises(RuntimeError, match="second"):
            (graph.square().sum() + y[n].square().sum()).backward()
        y[n].grad = None                       # (the other term's share)
        # a gradient kept with its graph is of use as it is
        call(*y).sum().backward(create_graph=True)
        assert torch.equal(y[n].grad.detach(), first)
        y[n].grad = None
