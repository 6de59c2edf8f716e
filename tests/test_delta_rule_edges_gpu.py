"""Rows and rates at the delta rule's edges, against the float64 recurrence within the bounds of
tests/_delta_rule_ref.py."""
import ctypes

import pytest
import torch

from mamba_amd import _native as nat
from mamba_amd.ops.delta_rule import delta_rule_fn
from tests._delta_rule_ref import bounds, check, recurrence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
NAMES = ("q", "k", "v", "g", "beta", "initial")


def make(B, L, H, G, K, V, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = {n: torch.randn(B, L, h, d, generator=gen) for n, h, d in (("q", G, K), ("k", G, K), ("v", H, V), ("dout", H, V))}
    x["k"] = x["k"] / torch.linalg.vector_norm(x["k"], dim=-1, keepdim=True)
    x = {n: t.to(dtype) for n, t in x.items()}
    x["g"] = -torch.rand(B, L, H, generator=gen) * 0.2
    x["beta"] = torch.sigmoid(torch.randn(B, L, H, generator=gen))
    x["initial"], x["dlast"] = (torch.randn(B, H, K, V, generator=gen) for _ in range(2))
    return {n: t.to(DEV) for n, t in x.items()}


def run(x):
    leaves = [x[n].detach().requires_grad_() for n in NAMES]
    out, last = delta_rule_fn(*leaves[:5], initial_state=leaves[5], return_last_state=True)
    got = {"out": out.detach(), "last": last.detach()}
    got.update(zip(["d" + n for n in NAMES], torch.autograd.grad([out, last], leaves, [x["dout"], x["dlast"]])))
    return got


def want_of(x):
    s = x["q"].shape[-1] ** -0.5
    want = recurrence(*(x[n] for n in ("q", "k", "v", "g", "beta")), s, x["initial"], None, x["dout"], x["dlast"])
    return want, bounds(want, x["v"].dtype, s)


def channels_first(t):
    """A (batch, heads, dim, seqlen) tensor of t's values."""
    y = torch.empty([t.shape[i] for i in (0, 2, 3, 1)], dtype=t.dtype, device=t.device)
    return y.copy_(t.permute(0, 2, 3, 1))


# One token: its stride says nothing of the row's width.
ONE = {
    "channels first": lambda t: channels_first(t).permute(0, 3, 1, 2),
    "stride 0": lambda t: t.contiguous().as_strided(t.shape, (t.stride(0), 0, t.stride(2), 1)),
    "stride 1": lambda t: t.contiguous().as_strided(t.shape, (t.stride(0), 1, t.stride(2), 1)),
    "far stride": lambda t: t.contiguous().as_strided(t.shape, (t.stride(0), 1 << 40, t.stride(2), 1)),
}


@TYPES
@pytest.mark.parametrize("shape", [(2, 1, 2, 2, 64, 64), (3, 1, 4, 2, 32, 48), (1, 1, 2, 1, 128, 128), (1, 1, 1, 1, 256, 72)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("stride", list(ONE))
def test_one_token_of_any_stride(stride, shape, dtype):
    x = make(*shape, dtype, seed=60 + sum(shape))
    want, room = want_of(x)
    plain = run(x)
    for n in ("q", "k", "v", "dout"):
        x[n] = ONE[stride](x[n])
        assert x[n].stride(-1) == 1 and not 3 <= x[n].stride(1) < 1 << 30
    got = run(x)
    for n, t in got.items():
        check(t, want[n], room[n], n)
        assert torch.equal(t, plain[n]), n


@TYPES
def test_gradient_through_a_permute(dtype):
    """A channels-first user: q, k and v come from a permute, and so does the gradient of out."""
    x = make(2, 1, 2, 2, 64, 64, dtype, seed=61)
    first = [channels_first(x[n]).requires_grad_() for n in ("q", "k", "v")]
    rest = [x[n].detach().requires_grad_() for n in ("g", "beta", "initial")]
    out, last = delta_rule_fn(*(t.permute(0, 3, 1, 2) for t in first), *rest[:2], initial_state=rest[2], return_last_state=True)
    grads = torch.autograd.grad([out.permute(0, 2, 3, 1), last], first + rest, [channels_first(x["dout"]), x["dlast"]])
    want, room = want_of(x)
    for n, t in zip(NAMES, grads):
        check(t.permute(0, 3, 1, 2) if n in "qkv" else t, want["d" + n], room["d" + n], n)


@TYPES
@pytest.mark.parametrize("stride", [0, 1, 1 << 40])
def test_one_token_through_c(stride, dtype):
    """Every row of one token between guards, out's among them, whatever its token stride says."""
    B, H, G, K, V = 2, 2, 1, 64, 64
    x = make(B, 1, H, G, K, V, dtype, seed=62)
    want = delta_rule_fn(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"])
    out = torch.full((B + 2, 1, H, V), 7.0, dtype=dtype, device=DEV)
    a = nat.DeltaRuleArgs(batch=B, seqlen=1, heads=H, groups=G, d_key=K, d_value=V, scale=K ** -0.5,
                          dtype={F32: nat.SS_F32, BF16: nat.SS_BF16, F16: nat.SS_F16}[dtype])
    for n, t in [(n, x[n]) for n in ("q", "k", "v", "g", "beta")] + [("out", out[1:-1])]:
        setattr(a, n, t.data_ptr())
        for d, s in (("batch", t.stride(0)), ("len", stride), ("head", t.stride(2))):
            setattr(a, f"{n}_{d}_stride", s)
    a.initial_state = x["initial"].data_ptr()
    a.workspace_bytes = nat.load().ss_delta_rule_fwd_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=DEV)
    a.workspace = ws.data_ptr()
    rc = nat.load().ss_delta_rule_fwd(ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, nat.load().ss_last_error()
    assert torch.equal(out[1:-1], want) and bool((out[0] == 7).all()) and bool((out[-1] == 7).all())


TINY = (0.0, 1e-20, -1e-22, 2.0 ** -60, 1e-30, -0.0, 1e-42)


@TYPES
@pytest.mark.parametrize("shape", [(1, 200, 2, 2, 64, 64), (1, 700, 2, 1, 128, 96)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_tiny_rates(shape, dtype):
    """dv and dk of a token have the factor beta: zero where it is, and as small as it is where it is tiny.

    Relative to beta their errors are those of other tokens', but for the type's smallest values.  A matrix instruction
    takes an operand's term below 2^-126 for zero: dk sums, over the 64 tokens of a chunk, two products of a factor beta R
    or beta M, in up to 3 terms, with an element of q or k, and so loses up to 64 * 2 * 3 * 2^-126 of the largest element.
    """
    x = make(*shape, dtype, seed=63)
    for i, b in enumerate(TINY):
        x["beta"][0, 3 + i::29] = b
    want, room = want_of(x)
    got = run(x)
    for n, t in got.items():
        check(t, want[n], room[n], n)
    for n, group in (("dv", 1), ("dk", shape[2] // shape[3])):
        smallest = 2.0 ** -24 if dtype == F16 else 2.0 ** -133 if dtype == BF16 else 2.0 ** -149
        if n == "dk":
            smallest += 64 * 2 * 3 * 2.0 ** -126 * max(float(x[m].abs().max()) for m in "qk")
        for i, b in enumerate(TINY):
            t, w, r = (y[0, 3 + i::29].double().cpu() for y in (got[n], want[n], room[n]))
            if b == 0.0:
                assert not t.any(), (n, b)
            else:
                step = torch.finfo(dtype).eps
                assert bool(((t - w).abs() <= r * abs(b) * (1 + step) + step * w.abs() + group * smallest).all()), (n, b)
