"""What linear_attn_update writes: autograd sees that state and out changed."""
import pytest
import torch

from mamba_amd.ops.linear_attn import linear_attn_fn, linear_attn_update

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def inputs(seed=0, B=2, L=70, H=4, G=2, K=32, V=24):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*s):
        return torch.randn(s, generator=gen, device=DEV)

    return rand(B, L, G, K), rand(B, L, G, K), rand(B, L, H, V), -rand(B, L, H).abs(), rand(B, H, K, V)


def test_a_saved_state_that_advanced_is_refused():
    q, k, v, g, state = inputs()
    q.requires_grad_()
    out = linear_attn_fn(q, k, v, g, initial_state=state)
    linear_attn_update(state, q[:, 0].detach(), k[:, 0], v[:, 0], g[:, 0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_versions():
    q, k, v, g, state = inputs(1)
    out = torch.empty_like(v[:, 0])
    before = state._version, out._version, q._version
    linear_attn_update(state, q[:, 0], k[:, 0], v[:, 0], g[:, 0], out=out)
    assert state._version > before[0] and out._version > before[1] and q._version == before[2]


def test_inference_mode():
    """A state made in inference mode has no version to raise, inside it and outside."""
    q, k, v, g, state = inputs(2)
    want = linear_attn_update(state.clone(), q[:, 0], k[:, 0], v[:, 0], g[:, 0])
    with torch.inference_mode():
        held = state.clone()
        assert torch.equal(linear_attn_update(held, q[:, 0], k[:, 0], v[:, 0], g[:, 0]), want)
        held.copy_(state)
    assert torch.equal(linear_attn_update(held, q[:, 0], k[:, 0], v[:, 0], g[:, 0]), want)


def test_overlapping_states_are_refused():
    q, k, v, g, state = inputs(3)
    t = q[:, 0], k[:, 0], v[:, 0], g[:, 0]
    for bad in (state[:1].expand_as(state), state[:, :1].expand_as(state)):
        before = bad.clone()
        with pytest.raises(ValueError, match="state's elements overlap"):
            linear_attn_update(bad, *t)
        assert torch.equal(bad, before)
    with pytest.raises(ValueError, match="out's elements overlap"):
        linear_attn_update(state, *t, out=torch.empty_like(v[:1, 0]).expand(2, 4, 24))
    # rows apart, heads in the other order of memory, and one row whose stride is anything
    want = state.clone()
    linear_attn_update(want, *t)
    for held in (torch.zeros(4, 2, 32, 24, device=DEV).transpose(0, 1), torch.zeros(2, 9, 32, 24, device=DEV)[:, 1::2]):
        held.copy_(state)
        linear_attn_update(held, *t)
        assert torch.equal(held, want)
    one = state[:1].clone()
    linear_attn_update(one.as_strided(one.shape, (0, *one.stride()[1:])), *(x[:1] for x in t))
    assert torch.equal(one, want[:1])
