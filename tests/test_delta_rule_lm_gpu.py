"""DeltaRule and LinearAttnLM of DeltaRule mixers on the GPU: logits and gradients against the formulas in
float64, a prompt and single tokens, rows of different lengths, autocast, a decode step in a graph and the example."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

from mamba_amd.models.linear_attn_lm import LinearAttnLM, LinearAttnLMConfig
from mamba_amd.modules.delta_rule import DeltaRule

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def model_of(dtype=torch.float32, **kw):
    torch.manual_seed(0)
    cfg = LinearAttnLMConfig(**{"vocab_size": 50, "model_dim": 48, "num_layers": 2, "head_dim": 16, "n_groups": 3, "mixer": "delta_rule", **kw})
    m = LinearAttnLM(cfg, device=DEV, dtype=dtype)
    assert all(type(x) is DeltaRule for x in m.mixers)
    for p in list(m.pre) + list(m.post) + [x.norm for x in m.mixers]:
        torch.nn.init.normal_(p, std=0.1)
    return m


def plain_logits(m, ids):
    """The model in float64 from its formulas, differentiable, on the CPU."""
    P = {n: p.detach().double().cpu().requires_grad_() for n, p in m.named_parameters()}
    eps = m.config.eps

    def rms(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * (1 + w)

    s = P["embedding.weight"][ids.cpu()]
    normed = rms(s, P["pre.0"])
    B, L, _ = s.shape
    for i, mix in enumerate(m.mixers):
        w = {n.split(".", 2)[2]: t for n, t in P.items() if n.startswith(f"mixers.{i}.")}
        qk, v, z, dt, b = (normed @ w["input_proj.weight"].T).split(mix.sizes, -1)
        r = mix.n_heads // mix.n_groups
        qk = qk.reshape(B, L, 2, mix.n_groups, mix.key_dim)
        qk = qk * torch.rsqrt(qk.square().sum(-1, keepdim=True) + eps)
        q, k = (t.repeat_interleave(r, 2) for t in qk.unbind(2))
        v = v.reshape(B, L, mix.n_heads, mix.head_dim)
        a = torch.exp(-torch.exp(w["log_A"]) * F.softplus(dt + w["dt_bias"]))
        beta = torch.sigmoid(b)
        S, outs = torch.zeros(B, mix.n_heads, mix.key_dim, mix.head_dim, dtype=torch.float64), []
        for t in range(L):
            S = S * a[:, t, :, None, None]
            e = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * S).sum(2))
            S = S + k[:, t, :, :, None] * e[:, :, None, :]
            outs.append((q[:, t, :, :, None] * S).sum(2) * mix.key_dim ** -0.5)
        o = torch.stack(outs, 1)
        y = rms(o, w["norm"].view(mix.n_heads, mix.head_dim)).flatten(2) * F.silu(z)
        s = s + P[f"scale.{i}"] * rms(y @ w["output_proj.weight"].T, P[f"post.{i}"])
        normed = rms(s, P[f"pre.{i + 1}"])
    return normed @ P["lm_head.weight"].T, P


def test_against_the_formulas():
    m = model_of()
    ids = torch.randint(0, 50, (2, 70), device=DEV)
    want, P = plain_logits(m, ids)
    got = m(ids)
    # fp32 through two layers of products over up to 192 terms: 2^-24 times a few thousand, of order-one values
    tol = 2.0 ** -12
    assert (got.double().cpu() - want).abs().max() <= tol * want.abs().max()
    up = torch.randn(want.shape, dtype=torch.float64)
    want.backward(up)
    got.backward(up.float().to(DEV))
    for n, p in m.named_parameters():
        w = P[n].grad
        assert (p.grad.double().cpu() - w).abs().max() <= tol * w.abs().max(), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_prompt_and_steps_agree(dtype):
    m = model_of(dtype)
    ids = torch.randint(0, 50, (3, 45), device=DEV)
    with torch.no_grad():
        whole = m(ids).float()
        states = m.allocate_states(3)
        first = m(ids[:, :30], states=states).float()
        rest = torch.stack([m.step(ids[:, t], states) for t in range(30, 45)], 1).float()
    got = torch.cat([first, rest], 1)
    # two orders of summation in fp32; in bf16 the layers' outputs are rounded (2^-8) about ten times
    tol = 2.0 ** -12 if dtype == torch.float32 else 10 * 2.0 ** -8
    assert (got - whole).abs().max() <= tol * whole.abs().max()


def test_rows_of_different_lengths():
    m = model_of()
    ids = torch.randint(0, 50, (3, 40), device=DEV)
    n = torch.tensor([40, 1, 17], device=DEV)
    with torch.no_grad():
        states = m.allocate_states(3)
        got = m(ids, lengths=n, states=states)
        for b in range(3):
            alone_states = m.allocate_states(1)
            alone = m(ids[b:b + 1, :n[b]], states=alone_states)
            assert (got[b, :n[b]] - alone[0]).abs().max() <= 2.0 ** -12 * alone.abs().max()
            for s, a in zip(states, alone_states):
                assert (s[b] - a[0]).abs().max() <= 2.0 ** -12 * a.abs().max()
        answers = m.generate(ids, 5, lengths=n)
        assert torch.equal(m.generate(ids[2:3, :17], 5)[0], answers[2])


def test_step_in_a_graph():
    m = model_of(torch.bfloat16)
    ids = torch.randint(0, 50, (4, 3), device=DEV)
    states, held = m.allocate_states(4), ids[:, 0].clone()
    want = [m.step(ids[:, t], states).clone() for t in range(3)]
    states = m.allocate_states(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(held, states)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.step(held, states)
    for turn in range(2):
        for s in states:
            s.zero_()
        for t in range(3):
            held.copy_(ids[:, t])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want[t]), (turn, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_autocast(dtype):
    torch.manual_seed(0)
    m = LinearAttnLM(LinearAttnLMConfig(vocab_size=30, model_dim=48, num_layers=2, head_dim=16, mixer="delta_rule"), device=DEV)
    ids = torch.randint(0, 30, (2, 40), device=DEV)
    want = m(ids)
    with torch.autocast("cuda", dtype):
        got = m(ids)
    # products of order-one rows rounded to dtype about ten times on the way
    assert (got.float() - want).abs().max() <= 10 * torch.finfo(dtype).eps * want.abs().max()
    got.float().square().sum().backward()
    assert all(p.grad.dtype == torch.float32 and p.grad.isfinite().all() for p in m.parameters())


def test_unknown_mixers_are_refused():
    with pytest.raises(ValueError, match="mixer"):
        LinearAttnLM(LinearAttnLMConfig(mixer="other"), device=DEV)


def test_the_example_runs():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_linear_attn_lm.py")
    spec = importlib.util.spec_from_file_location("train_linear_attn_lm", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    m, losses = ex.train(steps=3, symbols=4, length=6, log=lambda _: None, mixer="delta_rule")
    assert len(losses) == 3 and all(p.isfinite().all() for p in m.parameters())
    assert type(m.mixers[0]) is DeltaRule
