"""The gradient of a log decay relative to the decay itself: d out / d g_t carries
the factor exp(g_t), and so does its error where the decay is strong."""
import ctypes
import math

import pytest
import torch

from mamba_amd import _native as nat
from mamba_amd.ops.linear_attn import linear_attn_fn
from tests._linear_attn_ref import recurrence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
STRONG = -12 * math.log(2.0)         # below it a decay's gradient is summed by itself


def segment(B, L, H, G, K, V):
    a = nat.LinearAttnArgs()
    a.batch, a.seqlen, a.heads, a.groups, a.d_key, a.d_value, a.dtype = B, L, H, G, K, V, nat.SS_F32
    a.q = a.k = a.v = a.g = 1 << 20
    n = nat.load().ss_linear_attn_segment(ctypes.byref(a))
    assert n > 0
    return n


def room(x, scale):
    """How far dg may be off, from the recurrence on absolute values (m): C 2^-24 of what is summed, C = d_key +
    d_value + 64 + L / 64 + 32 as for the other gradients, and a token for every product of a segment (its
    sums and the factors of its decays).  A strong decay's sum has its own factor in every term: exp(g) <|S|, |R|>.  Any other
    starts at the next strong decay or the segment's end and adds the tokens' |q dq| + |k dk| up to there."""
    a = {n: None if x[n] is None else x[n].detach().double().cpu().abs() for n in ("q", "k", "v", "initial", "dout", "dlast")}
    m = recurrence(a["q"], a["k"], a["v"], x["g"], scale, a["initial"], x["lengths"], a["dout"], a["dlast"])
    B, L, G, K = x["q"].shape
    H, V = x["v"].shape[2:]
    n = segment(B, L, H, G, K, V)
    r = H // G
    g = x["g"].detach().double().cpu().expand(B, L, H)
    if r > 1:      # |q| |dq| of each head by itself: from the recurrence with every head a key of its own
        wide = recurrence(a["q"].repeat_interleave(r, 2), a["k"].repeat_interleave(r, 2), a["v"], x["g"], scale, a["initial"], x["lengths"],
                          a["dout"], a["dlast"])
    else:
        wide = m
    q, k = a["q"].repeat_interleave(r, 2), a["k"].repeat_interleave(r, 2)
    terms = (q * wide["dq"]).sum(-1) + (k * wide["dk"]).sum(-1)
    strong = g < STRONG
    total = torch.zeros_like(terms)
    for t in range(L - 1, -1, -1):
        if t + 1 == L or (t + 1) % n == 0:
            start = m["dg"][:, t + 1] if t + 1 < L else (m["dg"][:, t] * 0 + _end(m, a, x))
        else:
            start = torch.where(strong[:, t + 1], m["dg"][:, t + 1], total[:, t + 1])
        total[:, t] = start + terms[:, t]
    c = (K + V + 64 + L / 64 + 32 + n) * 2.0 ** -24
    return c * torch.where(strong, m["dg"], total), strong


def _end(m, a, x):
    """<|S|, |dS|> after the last token"""
    return 0.0 if a["dlast"] is None else (m["last"] * a["dlast"]).sum((2, 3))


def make(B, L, H, G, K, V, dtype, seed, initial=True, lengths=None):
    gen = torch.Generator().manual_seed(seed)
    x = {n: torch.randn(B, L, h, d, generator=gen).to(dtype) for n, h, d in (("q", G, K), ("k", G, K), ("v", H, V), ("dout", H, V))}
    x["g"] = -torch.rand(B, L, H, generator=gen) * 0.1
    x["initial"] = torch.randn(B, H, K, V, generator=gen) if initial else None
    x["dlast"] = torch.randn(B, H, K, V, generator=gen) if initial else None
    x["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    x["pick"] = torch.rand(B, L, H, generator=gen)
    return {n: None if t is None else t.to(DEV) for n, t in x.items()}


def compare(x):
    leaves = {n: x[n].detach().clone().requires_grad_() for n in ("q", "k", "v", "g", "initial") if x[n] is not None}
    o, last = linear_attn_fn(leaves["q"], leaves["k"], leaves["v"], leaves["g"], initial_state=leaves.get("initial"),
                             lengths=x["lengths"], return_last_state=True)
    outs, ups = ([o, last], [x["dout"], x["dlast"]]) if x["dlast"] is not None else ([o], [x["dout"]])
    got, = torch.autograd.grad(outs, [leaves["g"]], ups)
    got = got.double().cpu()
    scale = x["q"].shape[-1] ** -0.5
    want = recurrence(x["q"], x["k"], x["v"], x["g"], scale, x["initial"], x["lengths"], x["dout"], x["dlast"])["dg"]
    bound, strong = room(x, scale)
    if x["g"].dim() == 1:
        want, bound = want.sum((0, 1)), bound.sum((0, 1))
    bad = ~((got - want).abs() <= bound + torch.finfo(F32).tiny)
    assert not bad.any(), (int(bad.sum()), int((bad & strong).sum()) if bad.shape == strong.shape else None,
                           float(((got - want).abs() / (bound + 1e-300)).max()))
    return got


SHAPES = [(1, 1, 1, 1, 16, 16), (2, 70, 2, 2, 64, 64), (1, 200, 4, 2, 32, 24), (1, 130, 1, 1, 96, 130), (2, 1100, 2, 1, 20, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_some_strong_decays(shape, dtype):
    x = make(*shape, dtype, seed=sum(shape))
    for i, v in enumerate((-8.0, -10.0, -20.0, -60.0, -float("inf"), torch.finfo(F32).min)):
        x["g"][(x["pick"] >= 0.02 * i) & (x["pick"] < 0.02 * (i + 1))] = v
    got = compare(x)
    reset = torch.exp(x["g"]).cpu() == 0
    assert not got[reset].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("strength", [-7.0, -10.0, -20.0, -50.0])
def test_every_decay_strong(strength, dtype):
    x = make(2, 150, 2, 2, 64, 64, dtype, seed=3)
    x["g"] = x["g"] + strength
    compare(x)


@pytest.mark.parametrize("strength", [-10.0, -20.0, -float("inf")])
def test_one_strong_decay(strength):
    """One document boundary in a row; at segments' and chunks' borders too."""
    for t in (0, 1, 31, 32, 63, 64, 100, 149):
        x = make(1, 150, 2, 2, 64, 64, F32, seed=4)
        x["g"][0, t, 0] = strength
        compare(x)


def test_long_segments():
    """Enough rows that a segment is longest."""
    x = make(1600, 1100, 1, 1, 4, 4, F32, seed=5, lengths=[(13 * i) % 1101 for i in range(1600)])
    assert segment(1600, 1100, 1, 1, 4, 4) == 1024
    x["g"][x["pick"] < 0.003] = -15.0
    x["g"][x["pick"] > 0.999] = -float("inf")
    compare(x)


def test_one_strong_decay_per_head():
    x = make(2, 90, 4, 2, 32, 32, F32, seed=6)
    x["g"] = torch.tensor([-0.1, -9.0, -25.0, -float("inf")], device=DEV)
    got = compare(x)
    assert got[3] == 0


def test_lengths():
    x = make(4, 150, 2, 2, 48, 40, BF16, seed=7, lengths=[0, 1, 77, 150])
    x["g"][x["pick"] < 0.1] = -11.0
    compare(x)


def test_logarithm_of_a_factor():
    """g = log f: dg / f is the derivative in f, about <S, R> at a tiny f as at any other."""
    x = make(1, 80, 1, 1, 32, 32, F32, seed=8)
    f = torch.full((1, 80, 1), 0.9, device=DEV)
    f[0, 40] = 1e-9
    x["g"] = torch.log(f)
    got = compare(x)
    want = recurrence(x["q"], x["k"], x["v"], x["g"], 32 ** -0.5, x["initial"], None, x["dout"], x["dlast"])["dg"]
    assert abs(float(got[0, 40, 0] / want[0, 40, 0]) - 1) < 1e-3


def test_the_same_bits_every_run_and_captured():
    x = make(2, 300, 2, 2, 64, 64, BF16, seed=9)
    x["g"][x["pick"] < 0.05] = -13.0
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "initial")]

    def run():
        o = linear_attn_fn(*leaves[:4], initial_state=leaves[4])
        return torch.autograd.grad(o, leaves, x["dout"])

    want = run()
    for a, b in zip(run(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
