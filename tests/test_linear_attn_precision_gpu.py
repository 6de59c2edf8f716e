"""How near the linear attention's fp32 results are to the float64 recurrence, as
root mean squares and means over all of a result's elements.

A sum of n products in fp32 whose roundings are independent is off by about
2^-24 sqrt(n) of the root of its squared terms' sum (rms); n is at most d_key + d_value
+ 32 tokens of a chunk, and as many again for the factors and the chunks before.
Roundings to nearest have no sign: a sum of positive terms is off by less than half
a step (2^-24) on average.  Results kept in 16 bits are left out: their last rounding
hides the rest."""
import pytest
import torch

from mamba_amd.ops.linear_attn import linear_attn_fn
from tests._linear_attn_ref import recurrence
from tests.test_linear_attn_decay_grad_gpu import segment

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [(2, 300, 4, 4, 64, 64), (2, 515, 6, 2, 96, 80), (1, 400, 4, 2, 30, 128), (1, 1100, 2, 2, 160, 100)]


def run(shape, dtype, positive=False):
    B, L, H, G, K, V = shape
    gen = torch.Generator().manual_seed(sum(shape))
    rand = (lambda *s: torch.rand(s, generator=gen)) if positive else (lambda *s: torch.randn(s, generator=gen))
    x = {n: rand(B, L, h, d).to(dtype).to(DEV) for n, h, d in (("q", G, K), ("k", G, K), ("v", H, V), ("dout", H, V))}
    x["g"] = (-0.1 * torch.rand(B, L, H, generator=gen)).to(DEV)
    x["initial"], x["dlast"] = rand(B, H, K, V).to(DEV), rand(B, H, K, V).to(DEV)
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "initial")]
    out, last = linear_attn_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
    got = [out, last, *torch.autograd.grad([out, last], leaves, [x["dout"], x["dlast"]])]
    want = recurrence(x["q"], x["k"], x["v"], x["g"], K ** -0.5, x["initial"], None, x["dout"], x["dlast"])
    return x, {n: (t.detach().double().cpu(), want[n]) for n, t in zip(("out", "last", "dq", "dk", "dv", "dg", "dinitial"), got)
               if t.dtype == F32}


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_root_mean_squares(shape, dtype):
    B, L, H, G, K, V = shape
    x, res = run(shape, dtype)
    tol = 2.0 ** -24 * (2 * (K + V + 32)) ** 0.5
    for n, (got, want) in res.items():
        size = want
        if n == "dg":       # the sum of q dq - k dk from the token to its segment's end: the root of the squares' sum
            r, seg = H // G, segment(*shape)
            per_head = recurrence(x["q"].repeat_interleave(r, 2), x["k"].repeat_interleave(r, 2), x["v"], x["g"], K ** -0.5, x["initial"], None,
                                  x["dout"], x["dlast"])
            sq = sum((x[a].double().cpu().repeat_interleave(r, 2) * per_head["d" + a]).square().sum(-1) for a in ("q", "k"))
            size = torch.cat([s.flip(1).cumsum(1).flip(1) for s in sq.split(seg, 1)], 1)
            size = (size + want.square()).sqrt()
        off, rms = (got - want).square().mean().sqrt(), size.square().mean().sqrt()
        assert off <= tol * rms, (n, float(off / rms), tol)


@pytest.mark.parametrize("shape", [SHAPES[0], *SHAPES[2:]], ids=lambda s: "x".join(map(str, s)))
def test_roundings_have_no_sign(shape):
    _, res = run(shape, F32, positive=True)
    for n, (got, want) in res.items():
        if n != "dg":
            assert abs(float((got - want).mean() / want.mean())) <= 2.0 ** -24, n
