"""layer_norm_fn, unit_norm_fn and the LayerNorm module on the GPU against float64.

Bounds.  A sum of n numbers in fp32 is off by at most n 2^-24 of the sum of their sizes, here along trees and
lanes of at most 16 + 8 + 16 terms one after another: 64 2^-24 with the roundings around it covers each.  Let S be the
largest |s| of a row: its mean is off by 64 2^-24 S, so (s - m) by that, and what follows by
64 2^-24 (S r + |h|) a factor (r the reciprocal root, h the normalised element).  Weight gradients
add the same over rows.  A 16-bit result is rounded once more."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from mamba_amd.modules.layer_norm import LayerNorm
from mamba_amd.ops.layer_norm import layer_norm_fn
from mamba_amd.ops.unit_norm import unit_norm_fn
from tests._delta_rule_ref import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
U = 64 * 2.0 ** -24


def make(shape, dtype, seed=0, residual=True, bias=True, wdtype=None, shift=0.0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)

    def r(*s, t=dtype, mul=1.0, add=0.0):
        return (torch.randn(s, generator=gen) * mul + add).to(t).to(DEV)

    w = wdtype or dtype
    return {"x": r(*shape, mul=scale, add=shift), "weight": r(shape[-1], t=w, mul=0.3, add=1.0), "bias": r(shape[-1], t=w) if bias else None,
            "residual": r(*shape, mul=scale) if residual else None, "dout": r(*shape), "ds": r(*shape)}


def run(x, eps=1e-5, prenorm=True):
    leaves = {n: x[n].detach().requires_grad_() for n in ("x", "weight", "bias", "residual") if x[n] is not None}
    o, s = layer_norm_fn(leaves["x"], leaves["weight"], leaves.get("bias"), leaves.get("residual"), eps, prenorm=True)
    got = {"out": o, "s": s}
    outs, ups = ([o, s], [x["dout"], x["ds"]]) if prenorm else ([o], [x["dout"]])
    for n, t in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups)):
        got["d" + n] = t
    return got


def compare(x, got, eps=1e-5, prenorm=True):
    t = x["x"].dtype
    d = {n: None if v is None else v.detach().double().cpu() for n, v in x.items()}
    s = (x["x"].float() + x["residual"].float()).to(t).double().cpu() if x["residual"] is not None else d["x"]
    m = s.mean(-1, keepdim=True)
    r = (((s - m) ** 2).mean(-1, keepdim=True) + eps) ** -0.5
    h = (s - m) * r
    big = s.abs().amax(-1, keepdim=True) * r                     # S r
    eh = U * (big + h.abs()) * (1 + big)                         # (r itself by 2^-24 64 S r of its size)
    o = d["dout"] * d["weight"]
    m0, m1 = o.mean(-1, keepdim=True), (o * h).mean(-1, keepdim=True)
    dx = r * (o - m0 - h * m1) + (d["ds"] if prenorm else 0.0)
    oa = o.abs().mean(-1, keepdim=True)
    ha = h.abs().amax(-1, keepdim=True)
    edx = r * (U * (1 + big) * (o.abs() + oa + h.abs() * oa * ha) + eh * oa * ha + h.abs() * oa * eh.amax(-1, keepdim=True)) + U * d["ds"].abs()
    rows = list(range(s.dim() - 1))
    want = {"out": (h * d["weight"] + (d["bias"] if d["bias"] is not None else 0.0), eh * d["weight"].abs() + U * (h * d["weight"]).abs()
                    + (U * d["bias"].abs() if d["bias"] is not None else 0.0)),
            "s": (s, torch.zeros_like(s)), "dx": (dx, edx), "dresidual": (dx, edx),
            "dweight": ((d["dout"] * h).sum(rows), (d["dout"].abs() * (eh + U * h.abs())).sum(rows) * 4),
            "dbias": (d["dout"].sum(rows), U * d["dout"].abs().sum(rows) * 4)}
    for n, g in got.items():
        if n == "s":
            assert torch.equal(g, (x["x"] + x["residual"]) if x["residual"] is not None else x["x"])
        else:
            check(g, *want[n], n)


@TYPES
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (16, 768), (5, 1001), (2, 4, 64), (130, 512), (4100, 40), (7, 2048), (3, 4095),
                                   (2, 8192), (2, 16384), (3, 9001), (33, 1024)], ids=lambda s: "x".join(map(str, s)))
def test_layer_norm(shape, dtype):
    x = make(shape, dtype, seed=sum(shape))
    compare(x, run(x))


@TYPES
@pytest.mark.parametrize("residual,bias,prenorm", [(False, True, True), (False, False, True), (True, False, False), (False, True, False)])
def test_parts_left_out(residual, bias, prenorm, dtype):
    x = make((37, 200), dtype, seed=1, residual=residual, bias=bias)
    x["ds"] = x["ds"] if prenorm else torch.zeros_like(x["ds"])
    got = run(x, prenorm=prenorm)
    compare(x, got, prenorm=prenorm)
    w = x["weight"].clone().requires_grad_()
    alone, = torch.autograd.grad(layer_norm_fn(x["x"], w, x["bias"], x["residual"]), [w], x["dout"])
    assert torch.equal(alone, got["dweight"])


def test_only_the_stream():
    """The norm's output unused: what arrives at s passes through."""
    x = make((5, 100), F32, seed=2)
    a = x["x"].clone().requires_grad_()
    _, s = layer_norm_fn(a, x["weight"], x["bias"], x["residual"], prenorm=True)
    g, = torch.autograd.grad(s, [a], x["ds"])
    assert torch.equal(g, x["ds"])


def test_rows_far_from_zero():
    """The mean is off before squares are summed: rows of 1000 + N(0, 1) keep their spread."""
    x = make((64, 768), F32, seed=3, residual=False, shift=1000.0)
    got = run(x)
    compare(x, got)
    s = x["x"].double()
    want = torch.nn.functional.layer_norm(s, (768,), x["weight"].double(), x["bias"].double())
    # the mean's rounding (2^-24 of 1000, and its sum's) against a spread of 1, not the square's
    assert (got["out"].double() - want).abs().max() <= 1000 * 8 * 2.0 ** -24 * 1.3


def test_equal_rows():
    """A row of one value: no spread, the root is eps'."""
    x = make((4, 96), F32, seed=4, residual=False)
    x["x"] = torch.full_like(x["x"], 3.25)
    got = run(x)
    assert torch.equal(got["out"].detach(), x["bias"].expand(4, 96))
    compare(x, got)


@pytest.mark.parametrize("wdtype", [F32, BF16])
def test_weights_of_another_type(wdtype):
    x = make((40, 300), F16, seed=5, wdtype=wdtype)
    got = run(x)
    assert got["dweight"].dtype == got["dbias"].dtype == wdtype
    compare(x, got)


@TYPES
def test_layouts(dtype):
    x = make((6, 50, 96), dtype, seed=6)
    want = run(x)
    for change in (lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2], lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                   lambda t: t.repeat_interleave(2, -1)[..., ::2]):
        y = {n: change(t) if t is not None and t.dim() == 3 else t for n, t in x.items()}
        got = run(y)
        for n in want:
            assert torch.equal(got[n], want[n]), n
    y = {**x, "x": x["x"][:1].expand_as(x["x"])}
    compare(y, run(y))


def test_infinities_stay_in_their_row():
    x = make((9, 130), BF16, seed=7)
    want = run(x)
    x["x"] = x["x"].clone()
    x["x"][3, 5], x["x"][6, 0] = float("nan"), float("inf")
    got = run(x)
    rows = [0, 1, 2, 4, 5, 7, 8]
    for n in ("out", "s", "dx"):
        assert torch.equal(got[n][rows], want[n][rows]) and not got[n][3].isfinite().all() and not got[n][6].isfinite().all()


@pytest.mark.parametrize("shape", [(0, 8), (3, 0), (2, 0, 8)])
def test_empty(shape):
    x = make(shape, F32)
    got = run(x)
    assert got["out"].shape == got["dx"].shape == shape and not got["dweight"].any() and not got["dbias"].any()


def test_bits_streams_graphs():
    x, y = make((300, 768), BF16, seed=8), make((300, 768), BF16, seed=9)
    want = [run(x), run(y)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(x)
    torch.cuda.current_stream().wait_stream(side)
    for n in again:
        assert torch.equal(again[n], want[0][n]), n
    held = {n: t.clone() for n, t in x.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(held)
    for turn in (1, 0, 1):
        for n, t in (x, y)[turn].items():
            held[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        eager = run((x, y)[1 - turn])
        for n in got:
            assert torch.equal(got[n], want[turn][n]) and torch.equal(eager[n], want[1 - turn][n]), (turn, n)


def test_results_change_in_place():
    x = make((4, 64), F32, seed=10)
    a = x["x"].clone().requires_grad_()
    o, s = layer_norm_fn(a, x["weight"], x["bias"], x["residual"], prenorm=True)
    o.mul_(2.0)
    g, = torch.autograd.grad(o, [a], x["dout"])
    b = x["x"].clone().requires_grad_()
    h, = torch.autograd.grad(layer_norm_fn(b, x["weight"], x["bias"], x["residual"]), [b], x["dout"] * 2)
    assert torch.equal(g, h)


@TYPES
def test_module(dtype):
    torch.manual_seed(0)
    for bias in (True, False):
        m = LayerNorm(96, bias=bias, device=DEV, dtype=dtype)
        with torch.no_grad():
            m.weight.uniform_(0.5, 1.5)
        x = make((10, 96), dtype, seed=11)
        o, s = m(x["x"], x["residual"], prenorm=True)
        x["weight"], x["bias"] = m.weight.detach(), m.bias.detach() if bias else None
        compare(x, {"out": o, "s": s})
        c = LayerNorm(96, bias=bias, dtype=dtype)
        c.load_state_dict(m.state_dict())
        oc, sc = c(x["x"].cpu(), x["residual"].cpu(), prenorm=True)
        compare(x, {"out": oc.to(DEV), "s": sc.to(DEV)})


def test_refusals():
    x = make((4, 32), F32, seed=12)
    for bad, msg in (({"weight": x["weight"][:8]}, "weight must be"), ({"bias": x["bias"].cpu()}, "bias is on"),
                     ({"residual": x["residual"].half()}, "residual must match"), ({"x": x["x"].double()}, "dtype"), ({"x": x["x"].cpu()}, "ROCm"),
                     ({"weight": x["weight"].long()}, "float tensor")):
        y = {**x, **bad}
        with pytest.raises(ValueError, match=msg):
            layer_norm_fn(y["x"], y["weight"], y["bias"], y["residual"])
    with pytest.raises(ValueError, match="eps"):
        layer_norm_fn(x["x"], x["weight"], eps=-1.0)
    with pytest.raises(ValueError, match="16384"):
        w = torch.zeros(16385, device=DEV)
        layer_norm_fn(torch.zeros(1, 16385, device=DEV), w)
    names = ("x", "weight", "bias", "residual")
    for n in names:
        with fwad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            y = {**x, n: fwad.make_dual(x[n], x[n])}
            layer_norm_fn(*(y[m] for m in names))
        y = {**x, n: x[n].clone().requires_grad_()}
        g, = torch.autograd.grad(layer_norm_fn(*(y[m] for m in names)).sum(), [y[n]], create_graph=True)
        with pytest.raises(RuntimeError, match="second"):
            (g.square().sum() + y[n].square().sum()).backward()


# -------------------------------------------------------------- unit norm --
def unit_want(x, dout, eps):
    x, dout = x.detach().double().cpu(), dout.double().cpu()
    r = (x.square().sum(-1, keepdim=True) + eps) ** -0.5
    y = x * r
    yd, ya = (y * dout).sum(-1, keepdim=True), (y * dout).abs().sum(-1, keepdim=True)
    return {"out": (y, U * y.abs()), "dx": (r * (dout - y * yd), U * r * (dout.abs() + y.abs() * ya * 3))}


def unit_run(x, dout, eps=1e-6):
    a = x.detach().requires_grad_()
    o = unit_norm_fn(a, eps)
    return {"out": o, "dx": torch.autograd.grad(o, [a], dout)[0]}


@TYPES
@pytest.mark.parametrize("shape", [(1,), (5,), (3, 1), (2, 3, 7), (4, 5, 6, 64), (300, 48, 64), (64, 32, 128), (7, 200), (2, 300),
                                   (3, 2, 1000), (2, 5000), (2, 16384), (9, 3, 33)], ids=lambda s: "x".join(map(str, s)))
def test_unit_norm(shape, dtype):
    gen = torch.Generator().manual_seed(sum(shape))
    x, d = (torch.randn(shape, generator=gen).to(dtype).to(DEV) for _ in range(2))
    want = unit_want(x, d, 1e-6)
    for n, t in unit_run(x, d).items():
        check(t, *want[n], n)


@TYPES
def test_unit_norm_layouts(dtype):
    gen = torch.Generator().manual_seed(20)
    row = torch.randn(2, 30, 9 * 40 + 3, generator=gen).to(dtype).to(DEV)
    x = row[..., 3:3 + 8 * 40].view(2, 30, 8, 40)               # heads in a projection's output
    d = torch.randn(2, 30, 8, 40, generator=gen).to(dtype).to(DEV)
    want = unit_run(x.contiguous(), d)
    for a, b in ((x, d), (x.transpose(1, 2).contiguous().transpose(1, 2), d), (x, d.transpose(1, 2).contiguous().transpose(1, 2)),
                 (x.repeat_interleave(2, -1)[..., ::2], d.repeat_interleave(2, -1)[..., ::2])):
        got = unit_run(a, b)
        for n in want:
            assert torch.equal(got[n], want[n]), n
    one = unit_run(x[:, :1].expand(2, 30, 8, 40), d[:1, :1, :1].expand(2, 30, 8, 40))
    first = unit_run(x[:, :1].expand(2, 30, 8, 40).contiguous(), d[:1, :1, :1].expand(2, 30, 8, 40).contiguous())
    for n in one:
        assert torch.equal(one[n], first[n])
    q, k = unit_norm_fn(x).chunk(2, -2)
    assert torch.equal(q, want["out"][:, :, :4]) and torch.equal(k, want["out"][:, :, 4:])


def test_unit_norm_ends():
    """Rows of zeros, very small and large ones, infinities in one row."""
    x = torch.randn(6, 64, device=DEV)
    x[0], x[1], x[2], x[3, 7] = 0.0, x[1] * 1e-15, x[2] * 1e15, float("inf")
    d = torch.randn(6, 64, device=DEV)
    got, want = unit_run(x, d), unit_want(x, d, 1e-6)
    keep = [0, 1, 2, 4, 5]
    for n in got:
        check(got[n][keep], want[n][0][keep], want[n][1][keep], n)
        assert not got[n][3].isfinite().all()
    for shape in ((0, 4, 8), (3, 0, 8), (3, 4, 0)):
        e = torch.zeros(shape, device=DEV)
        assert unit_run(e, e)["dx"].shape == shape


def test_unit_norm_graphs_and_refusals():
    x, d = torch.randn(64, 8, 64, device=DEV), torch.randn(64, 8, 64, device=DEV)
    want = unit_run(x, d)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = unit_run(held, d)
    for _ in range(3):
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for n in got:
            assert torch.equal(got[n], want[n]), n
        held.zero_()
    with pytest.raises(ValueError, match="dtype"):
        unit_norm_fn(x.double())
    with pytest.raises(ValueError, match="ROCm"):
        unit_norm_fn(x.cpu())
    with pytest.raises(ValueError, match="eps"):
        unit_norm_fn(x, eps=-1.0)
    with pytest.raises(ValueError, match="16384"):
        unit_norm_fn(torch.zeros(1, 16385, device=DEV))
    with fwad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        unit_norm_fn(fwad.make_dual(x, x))
    a = x.clone().requires_grad_()
    g, = torch.autograd.grad(unit_norm_fn(a).sum(), [a], create_graph=True)
    with pytest.raises(RuntimeError, match="second"):
        (g.square().sum() + a.square().sum()).backward()
