"""The norms' gradients for rows far from one: a reciprocal root near the ends
of fp32's range, whose cube lies outside it."""
import pytest
import torch

from mamba_amd.ops.block_norm import block_norm_fn, gated_rms_norm_fn
from tests._block_norm_ref import border, check, heads

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16 = torch.float32, torch.bfloat16
SIZES = [1e-15, 1e-13, 1e13, 1e15]


def rand(gen, *shape, dtype=F32, mul=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * mul).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("both", [False, True], ids=["x", "x and residual"])
def test_border(size, dtype, both):
    gen = torch.Generator().manual_seed(1)
    x = {"x": rand(gen, 6, 96, dtype=dtype, mul=size), "res": rand(gen, 6, 96, dtype=dtype, mul=size if both else 1.0),
         "post": rand(gen, 96, mul=0.2), "pre": rand(gen, 96, mul=0.2), "gate": rand(gen, 6, 96, dtype=dtype), "scale": rand(gen, 96)}
    if both:                                 # (s of x's size: the scale carries it)
        x["scale"] = x["scale"] * size
    up = {"dout": rand(gen, 6, 96, dtype=dtype), "ds": rand(gen, 6, 96, dtype=dtype, mul=1.0 / size if both else 1.0)}
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    out, s = block_norm_fn(leaves["x"], leaves["res"], leaves["post"], leaves["pre"], gate=leaves["gate"], scale=leaves["scale"], eps=0.0)
    got = {"out": out, "s": s}
    for n, t in zip(leaves, torch.autograd.grad([out, s], list(leaves.values()), [up["dout"], up["ds"]])):
        got["d" + n] = t
    want, room = border(**x, eps=0.0, **up)
    for n, t in got.items():
        check(t, want[n], room[n], n)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n", [32, 600])
def test_heads(size, dtype, n):
    gen = torch.Generator().manual_seed(2)
    x = {"x": rand(gen, 5, 3 * n, dtype=dtype, mul=size), "gate": rand(gen, 5, 3 * n, dtype=dtype), "w": rand(gen, 3 * n, mul=0.2)}
    dout = rand(gen, 5, 3 * n, dtype=dtype)
    leaves = {k: t.clone().requires_grad_() for k, t in x.items()}
    out = gated_rms_norm_fn(leaves["x"], leaves["gate"], leaves["w"], n_groups=3, eps=0.0)
    got = {"out": out}
    for k, t in zip(("dx", "dgate", "dweight"), torch.autograd.grad(out, list(leaves.values()), dout)):
        got[k] = t
    want, room = heads(x["x"], x["gate"], x["w"], 3, 0.0, dout)
    for k, t in got.items():
        check(t, want[k], room[k], k)
