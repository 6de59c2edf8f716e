"""LinearAttnLM with fp32 parameters under autocast: 16-bit products beside an fp32 residual stream."""
import pytest
import torch

from mamba_amd.models.linear_attn_lm import LinearAttnLM, LinearAttnLMConfig

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_autocast(dtype):
    torch.manual_seed(0)
    m = LinearAttnLM(LinearAttnLMConfig(vocab_size=30, model_dim=48, num_layers=2, head_dim=16), device=DEV)
    ids = torch.randint(0, 30, (2, 40), device=DEV)
    want = m(ids)
    want.square().sum().backward()
    plain = [p.grad.clone() for p in m.parameters()]
    m.zero_grad()
    with torch.autocast("cuda", dtype):
        got = m(ids)
        states = m.allocate_states(2)
        with torch.no_grad():
            m(ids[:, :30], states=states)
            steps = torch.stack([m.step(ids[:, t], states) for t in range(30, 40)], 1)
    # products of order-one rows rounded to dtype about ten times on the way
    tol = 10 * torch.finfo(dtype).eps
    assert (got.float() - want).abs().max() <= tol * want.abs().max()
    assert (steps.float() - want[:, 30:]).abs().max() <= tol * want.abs().max()
    got.float().square().sum().backward()
    for p, g in zip(m.parameters(), plain):
        assert p.grad.dtype == torch.float32
        # (a gradient passes through as many roundings again, and the doubled error of the logits)
        assert (p.grad - g).norm() <= 4 * tol * g.norm()
