"""A token's update has no backward: it says so where a gradient would be lost."""
import pytest
import torch

from mamba_amd.models.linear_attn_lm import LinearAttnLM, LinearAttnLMConfig
from mamba_amd.ops.linear_attn import linear_attn_update

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("name", ["state", "q", "k", "v", "g"])
def test_update_refuses_to_drop_a_gradient(name):
    torch.manual_seed(0)
    x = {"state": torch.randn(2, 4, 16, 8, device=DEV), "q": torch.randn(2, 2, 16, device=DEV), "k": torch.randn(2, 2, 16, device=DEV),
         "v": torch.randn(2, 4, 8, device=DEV), "g": -torch.rand(2, 4, device=DEV)}
    want = linear_attn_update(**{**x, "state": x["state"].clone()})
    before = x["state"].clone()
    y = {**x, name: x[name].clone().requires_grad_()}
    with pytest.raises(ValueError, match="no backward"):
        linear_attn_update(**y)
    assert torch.equal(y["state"], before)
    with torch.no_grad():
        assert torch.equal(linear_attn_update(**y), want)


def test_steps_of_the_modules_carry_no_gradient():
    torch.manual_seed(0)
    m = LinearAttnLM(LinearAttnLMConfig(vocab_size=20, model_dim=32, num_layers=2, head_dim=16), device=DEV)
    ids = torch.randint(0, 20, (3, 6), device=DEV)
    states = m.allocate_states(3)
    m(ids, states=states)                      # with grad mode on: the states have a history
    logits = m.step(ids[:, 0], states)
    assert not logits.requires_grad and not m.mixers[0].step(torch.randn(3, 32, device=DEV), states[0]).requires_grad
    with torch.no_grad():
        again = m.allocate_states(3)
        m(ids, states=again)
        want = m.step(ids[:, 0], again)
    assert torch.equal(logits, want)
