"""linear_attn_fn and linear_attn_update on the GPU against the float64
recurrence, within bounds that tests/_linear_attn_ref.py derives."""
import pytest
import torch

from mamba_amd.ops.linear_attn import linear_attn_fn, linear_attn_update
from tests._linear_attn_ref import bounds, check, recurrence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(B, L, H, G, K, V, dtype, seed=0, per_head=False, initial=False, lengths=None, fast=False):
    gen = torch.Generator().manual_seed(seed)
    x = {n: torch.randn(B, L, h, d, generator=gen).to(dtype) for n, h, d in (("q", G, K), ("k", G, K), ("v", H, V), ("dout", H, V))}
    x["g"] = -torch.rand((H,) if per_head else (B, L, H), generator=gen) * (3.0 if fast else 0.2)
    x["initial"] = torch.randn(B, H, K, V, generator=gen) if initial else None
    x["dlast"] = torch.randn(B, H, K, V, generator=gen) if initial else None
    x["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return {n: None if t is None else t.to(DEV) for n, t in x.items()}


def run(x, grad=True, scale=None):
    leaves = {n: x[n].detach().requires_grad_(grad) for n in ("q", "k", "v", "g", "initial") if x[n] is not None}
    o, last = linear_attn_fn(leaves["q"], leaves["k"], leaves["v"], leaves["g"], scale=scale,
                             initial_state=leaves.get("initial"), lengths=x["lengths"], return_last_state=True)
    got = {"out": o, "last": last}
    if grad:
        outs, ups = ([o, last], [x["dout"], x["dlast"]]) if x["dlast"] is not None else ([o], [x["dout"]])
        for n, t in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups)):
            got["d" + n] = t
    return got


def compare(x, got, scale=None, what=""):
    s = x["q"].shape[-1] ** -0.5 if scale is None else scale
    a = (x["q"], x["k"], x["v"], x["g"], s, x["initial"], x["lengths"])
    grads = (x["dout"], x["dlast"]) if "dq" in got else ()
    want, room = recurrence(*a, *grads), bounds(*a, *grads)
    if x["g"].dim() == 1 and grads:
        want["dg"], room["dg"] = want["dg"].sum((0, 1)), room["dg"].sum((0, 1))
    for n, t in got.items():
        check(t, want[n], room[n], f"{what}{n}")


SHAPES = [
    # B, L, H, G, K, V
    (1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 16, 16), (1, 3, 2, 2, 7, 5), (2, 63, 2, 2, 64, 64), (1, 64, 3, 1, 64, 64),
    (2, 65, 2, 2, 64, 64), (1, 127, 4, 2, 32, 128), (1, 200, 2, 1, 128, 64), (2, 130, 2, 2, 96, 80), (1, 513, 2, 2, 20, 24),
    (1, 1030, 2, 2, 64, 64), (1, 150, 1, 1, 130, 200), (1, 140, 1, 1, 256, 256), (3, 90, 6, 2, 48, 33), (1, 2100, 1, 1, 16, 65),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(shape, dtype):
    x = make(*shape, dtype, seed=sum(shape), initial=shape[1] % 2 == 1)
    compare(x, run(x))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 300, 4, 2, 64, 64), (1, 77, 3, 3, 40, 72)], ids=lambda s: "x".join(map(str, s)))
def test_one_decay_per_head(shape, dtype):
    x = make(*shape, dtype, seed=3, per_head=True, initial=True)
    compare(x, run(x))


@pytest.mark.parametrize("shape", [(600, 1100, 2, 1, 8, 8), (1100, 70, 1, 1, 16, 16)], ids=lambda s: "x".join(map(str, s)))
def test_many_rows(shape):
    """Enough rows to fill the GPU: each is walked whole, through one segment or several."""
    lengths = [(7 * i) % (shape[1] + 1) for i in range(shape[0])]
    x = make(*shape, BF16, seed=30, initial=True, lengths=lengths)
    x["g"] = x["g"] * 0.1
    compare(x, run(x))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_lengths(dtype):
    x = make(6, 150, 4, 2, 64, 64, dtype, seed=4, initial=True, lengths=[0, 1, 64, 65, 150, 149])
    # what lies past a row's length is not read
    for b, n in enumerate(x["lengths"].tolist()):
        for t in ("q", "k", "v", "dout"):
            x[t][b, n:] = float("nan")
        x["g"][b, n:] = float("inf")
    got = run(x)
    y = dict(x)
    for b, n in enumerate(x["lengths"].tolist()):
        for t in ("q", "k", "v", "dout", "g"):
            y[t] = y[t].clone()
            y[t][b, n:] = 0.0
    compare(y, got)
    assert torch.equal(got["last"][0], x["initial"][0])


def test_lengths_beyond_the_row():
    x = make(2, 70, 2, 2, 32, 32, F32, seed=5, lengths=[1000, -3])
    compare(x, run(x))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decays_at_their_ends(dtype):
    """Resets (minus infinity, the type's lowest value), no decay and growth."""
    x = make(2, 200, 4, 4, 64, 64, dtype, seed=6, initial=True)
    lowest = torch.finfo(F32).min
    for b, t, h, v in ((0, 0, 0, -float("inf")), (0, 100, 0, -float("inf")), (0, 101, 0, lowest), (1, 63, 1, lowest),
                       (1, 64, 1, -float("inf")), (0, 199, 2, -float("inf")), (1, 10, 3, -90.0), (1, 130, 3, -200.0)):
        x["g"][b, t, h] = v
    x["g"][0, :, 3] = 0.0
    x["g"][1, :50, 0] = 0.05
    compare(x, run(x))


def test_strong_decays():
    x = make(2, 300, 2, 2, 64, 64, F32, seed=7, fast=True, initial=True)
    compare(x, run(x))


def test_a_later_token_reaches_no_earlier_one():
    """Infinities and NaN of a token leave the tokens before it alone."""
    for dtype in (F32, BF16, F16):
        x = make(1, 150, 2, 2, 64, 64, dtype, seed=8)
        want = run(x, grad=False)["out"]
        for t in (40, 130):
            for n, v in (("v", float("nan")), ("k", float("inf")), ("q", float("nan"))):
                y = dict(x)
                y[n] = x[n].clone()
                y[n][0, t, 0, 3] = v
                got = run(y, grad=False)["out"]
                assert torch.equal(got[0, :t], want[0, :t]), (dtype, t, n)
                assert torch.equal(got[0, :, 1], want[0, :, 1])
                assert not got[0, t, 0].isfinite().all()


LAYOUTS = {
    "one projection": lambda t, i: t,
    "heads first": lambda t, i: t.transpose(1, 2).contiguous().transpose(1, 2),
    "rows off 16 bytes": lambda t, i: torch.nn.functional.pad(t, (1, 2))[..., 1:-2],
    "every second column": lambda t, i: t.repeat_interleave(2, -1)[..., ::2],
    "batch broadcast": lambda t, i: t[:1].expand_as(t),
}


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_layouts(layout, dtype):
    x = make(2, 140, 4, 2, 64, 48, dtype, seed=9)
    if layout == "one projection":
        row = torch.cat([x[n].flatten(2) for n in ("q", "k", "v")], -1)
        q, k, v = row.split([128, 128, 192], -1)
        x["q"], x["k"], x["v"] = q.view(2, 140, 2, 64), k.view(2, 140, 2, 64), v.view(2, 140, 4, 48)
    else:
        for i, n in enumerate(("q", "k", "v", "dout")):
            x[n] = LAYOUTS[layout](x[n], i)
    x["g"] = x["g"].transpose(1, 2).contiguous().transpose(1, 2)
    compare(x, run(x))


def test_decays_in_the_rows_type():
    x = make(2, 100, 2, 2, 32, 32, BF16, seed=10)
    x["g"] = x["g"].bfloat16()
    got = run(x)
    assert got["dg"].dtype == BF16
    compare(x, got)


def test_only_some_gradients():
    x = make(1, 80, 2, 2, 32, 32, F32, seed=11, initial=True)
    full = run(x)
    v = x["v"].detach().requires_grad_()
    o = linear_attn_fn(x["q"], x["k"], v, x["g"], initial_state=x["initial"])
    alone, = torch.autograd.grad(o, [v], x["dout"])
    x["dlast"] = torch.zeros_like(x["dlast"])
    assert torch.equal(alone, run(x)["dv"])
    i = x["initial"].detach().requires_grad_()
    _, last = linear_attn_fn(x["q"], x["k"], x["v"], x["g"], initial_state=i, return_last_state=True)
    di, = torch.autograd.grad(last.sum(), [i])
    want = torch.exp(x["g"].double().sum(1))[..., None, None].expand_as(di).cpu()
    check(di, want, 200 * 2.0 ** -24 * want, "dinitial")
    assert full["out"].shape == o.shape


@pytest.mark.parametrize("shape", [(0, 5, 2, 2, 8, 8), (2, 0, 2, 1, 8, 8), (2, 5, 0, 1, 8, 8)], ids=["batch", "seqlen", "heads"])
def test_empty(shape):
    x = make(*shape, F32, initial=True)
    got = run(x)
    assert got["out"].shape == x["v"].shape and got["dq"].shape == x["q"].shape
    assert torch.equal(got["last"], x["initial"]) and torch.equal(got["dinitial"], x["dlast"])
    assert got["dg"].shape == x["g"].shape


def test_gradient_against_differences():
    """The derivative along a direction against central differences of the forward."""
    x = make(1, 130, 2, 1, 32, 32, F32, seed=12, initial=True)
    got = run(x)
    torch.manual_seed(0)
    w = x["dout"].double(), x["dlast"].double()

    def value(y):
        r = run(y, grad=False)
        return float((r["out"].double() * w[0]).sum() + (r["last"].double() * w[1]).sum())

    for n in ("q", "k", "v", "g", "initial"):
        d = torch.randn_like(x[n]) * (0.05 if n == "g" else 1.0)
        h = 2.0 ** -7
        up, down = (value({**x, n: x[n] + s * h * d}) for s in (1, -1))
        slope = float((got["d" + n].double() * d.double()).sum())
        # the third derivative's share (only g has one), and the forward's rounding over 2 h
        tol = 2.0 ** -12 * abs(slope) + 2.0 ** -20 / h * float((got["out"].double() * w[0]).abs().sum() + (got["last"].double() * w[1]).abs().sum())
        assert abs((up - down) / (2 * h) - slope) <= tol, n


def test_the_same_bits_every_run():
    x = make(2, 700, 4, 2, 64, 64, BF16, seed=13, initial=True)
    a, b = run(x), run(x)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_another_stream():
    x = make(1, 500, 2, 2, 64, 64, BF16, seed=14)
    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_captured():
    """Forward and backward in one graph, replayed on new inputs."""
    x = make(2, 300, 2, 2, 64, 64, BF16, seed=15, initial=True)
    y = make(2, 300, 2, 2, 64, 64, BF16, seed=16, initial=True)
    want = [run(x), run(y)]
    held = {n: None if t is None else t.clone() for n, t in x.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(held)
    for turn in (1, 0, 1):
        for n, t in (x, y)[turn].items():
            if t is not None:
                held[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for n in got:
            assert torch.equal(got[n], want[turn][n]), (turn, n)


def test_far_rows():
    """Row offsets past 2^31 elements."""
    far = torch.zeros((1 << 31) + 70 * 64 + 64, dtype=BF16, device=DEV)
    x = make(2, 70, 1, 1, 64, 64, BF16, seed=17)
    want = run(x)
    y = dict(x)
    y["v"] = far.as_strided((2, 70, 1, 64), (1 << 31, 64, 64, 1))
    y["v"].copy_(x["v"])
    got = run(y)
    for n in want:
        assert torch.equal(got[n], want[n]), n


# ------------------------------------------------------------ one token --
def _token(B, H, G, K, V, dtype, seed=0, per_head=False):
    x = make(B, 1, H, G, K, V, dtype, seed=seed, per_head=per_head, initial=True)
    return x, {n: x[n][:, 0] for n in ("q", "k", "v")} | {"g": x["g"] if per_head else x["g"][:, 0]}


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 24, 24, 64, 64), (64, 4, 2, 128, 128), (3, 6, 2, 96, 80), (2, 2, 1, 7, 33),
                                   (5, 2, 2, 256, 256), (2, 3, 3, 130, 6)], ids=lambda s: "x".join(map(str, s)))
def test_update(shape, dtype):
    x, t = _token(*shape, dtype, seed=sum(shape), per_head=shape[0] == 3)
    state = x["initial"].clone()
    o = linear_attn_update(state, t["q"], t["k"], t["v"], t["g"])
    compare(x, {"out": o[:, None], "last": state})


def test_update_continues_the_prompt():
    x = make(2, 100, 4, 2, 64, 64, BF16, seed=20)
    want, whole = linear_attn_fn(x["q"], x["k"], x["v"], x["g"], return_last_state=True)
    o, state = linear_attn_fn(x["q"][:, :90], x["k"][:, :90], x["v"][:, :90], x["g"][:, :90], return_last_state=True)
    out = torch.empty_like(x["v"][:, 0])
    for t in range(90, 100):
        r = linear_attn_update(state, x["q"][:, t], x["k"][:, t], x["v"][:, t], x["g"][:, t], out=out)
        assert r is out
        # both sides within the bounds of the recurrence: twice half a step of the larger plus the sums'
        assert (r.double() - want[:, t].double()).abs().max() <= 2.0 ** -7 * want[:, t].double().abs().max()
    assert (state - whole).abs().max() <= 2.0 ** -14 * whole.abs().max()


def test_update_resets_and_strides():
    x, t = _token(2, 4, 2, 64, 64, F32, seed=21)
    big = torch.zeros(2, 8, 64, 64, device=DEV)
    state = big[:, ::2]
    state.copy_(x["initial"])
    t["g"] = t["g"].clone()
    t["g"][0, 1], t["g"][1, 2] = -float("inf"), torch.finfo(F32).min
    x["g"] = t["g"][:, None]
    o = linear_attn_update(state, t["q"], t["k"], t["v"], t["g"])
    compare(x, {"out": o[:, None], "last": state})
    assert not big[:, 1::2].any()
    off = torch.zeros(2 * 4 * 64 * 64 + 1, device=DEV)[1:].view(2, 4, 64, 64)   # rows off 16 bytes
    off.copy_(x["initial"])
    o2 = linear_attn_update(off, t["q"], t["k"], t["v"], t["g"])
    compare(x, {"out": o2[:, None], "last": off})


def test_update_captured():
    x, t = _token(2, 4, 4, 64, 64, BF16, seed=22)
    state = x["initial"].clone()
    linear_attn_update(state, t["q"], t["k"], t["v"], t["g"])
    want = state.clone()
    state.copy_(x["initial"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        linear_attn_update(state, t["q"], t["k"], t["v"], t["g"])
    for _ in range(3):
        state.copy_(x["initial"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(state, want)
