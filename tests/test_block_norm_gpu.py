"""block_norm_fn, gated_rms_norm_fn and clip_grads on the GPU against float64,
within bounds that tests/_block_norm_ref.py derives."""
import math

import pytest
import torch

from mamba_amd.ops.block_norm import block_norm_fn, gated_rms_norm_fn
from mamba_amd.ops.clip_grads import clip_grads
from tests._block_norm_ref import border, check, heads

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]
TYPE_IDS = ["f32", "bf16", "bf16-wf32", "f16", "f16-wf32"]


def rand(gen, *shape, dtype=F32, mul=1.0):
    return (torch.randn(shape, generator=gen) * mul).to(dtype).to(DEV)


def make_border(rows, dim, dtype, wtype, gate=True, vec=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return {"x": rand(gen, rows, dim, dtype=dtype), "res": rand(gen, rows, dim, dtype=dtype, mul=2.0),
            "post": rand(gen, dim, dtype=wtype, mul=0.2), "pre": rand(gen, dim, dtype=wtype, mul=0.2),
            "gate": rand(gen, rows, dim, dtype=dtype, mul=2.0) if gate else None,
            "scale": rand(gen, dim, dtype=wtype) if vec else 0.5}, \
        {"dout": rand(gen, rows, dim, dtype=dtype), "ds": rand(gen, rows, dim, dtype=dtype)}


def run_border(x, up=None):
    leaves = {n: t.detach().requires_grad_(up is not None) if isinstance(t, torch.Tensor) else t for n, t in x.items()}
    o, s = block_norm_fn(leaves["x"], leaves["res"], leaves["post"], leaves["pre"], gate=leaves["gate"], scale=leaves["scale"], eps=EPS)
    got = {"out": o, "s": s}
    if up is not None:
        names = [n for n, t in leaves.items() if isinstance(t, torch.Tensor)]
        outs = [(o, up["dout"]), (s, up["ds"])]
        outs = [p for p in outs if p[1] is not None]
        for n, t in zip(names, torch.autograd.grad([p[0] for p in outs], [leaves[n] for n in names], [p[1] for p in outs])):
            got["d" + n] = t
    return got


def compare_border(x, got, up=None, what=""):
    up = up or {"dout": None, "ds": None}
    y = {n: t if isinstance(t, torch.Tensor) or t is None else torch.tensor(t) for n, t in x.items()}
    want, room = border(**y, eps=EPS, **up)
    for n, t in got.items():
        check(t, want[n], room[n], what + n)


SHAPES = [(1, 1), (3, 7), (5, 64), (2, 65), (4, 511), (3, 512), (9, 513), (7, 768), (2, 1001), (6, 1024), (3, 1025), (2, 2048),
          (3, 2050), (2, 4096), (2, 5003), (1, 8192), (2, 9001), (1, 16384)]


@pytest.mark.parametrize("types", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_border(shape, types):
    x, up = make_border(*shape, *types, gate=shape[0] != 2, vec=shape[0] != 3, seed=sum(shape))
    compare_border(x, run_border(x), what="no grad ")
    compare_border(x, run_border(x, up), up)


@pytest.mark.parametrize("types", TYPES[:3], ids=TYPE_IDS[:3])
def test_border_many_rows(types):
    x, up = make_border(5000, 100, *types, seed=1)
    compare_border(x, run_border(x, up), up)


@pytest.mark.parametrize("only", ["dout", "ds"])
def test_border_one_gradient(only):
    x, up = make_border(20, 96, F32, F32, seed=2)
    up = {n: t if n == only else None for n, t in up.items()}
    compare_border(x, run_border(x, up), up)


def test_border_cancelling_sum():
    """s far smaller than its terms: the bound grows with them, and holds."""
    x, up = make_border(40, 200, F32, F32, gate=False, vec=False, seed=3)
    t = border(**{**x, "scale": torch.tensor(0.5)}, eps=EPS)[0]["s"] - x["res"].double().cpu()
    x["res"] = (-t + 1e-3 * torch.randn(t.shape, dtype=torch.float64)).float().to(DEV)
    compare_border(x, run_border(x, up), up)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_border_layouts(dtype):
    x, up = make_border(24, 80, dtype, dtype, seed=4)
    wide = torch.zeros(24, 200, dtype=dtype, device=DEV)
    for i, n in enumerate(("x", "gate")):                    # slices of one projection, off 16 bytes
        wide[:, 1 + 100 * i:81 + 100 * i] = x[n]
        x[n] = wide[:, 1 + 100 * i:81 + 100 * i]
    x["res"] = x["res"].t().contiguous().t()                 # columns apart
    up["dout"] = up["dout"][:1].expand(24, 80)
    compare_border(x, run_border(x, up), up)
    y = {n: t.view(2, 3, 4, 80) if n in ("x", "res", "gate") and t.is_contiguous() else t for n, t in x.items()}
    y["x"], y["res"], y["gate"] = (x[n].contiguous().view(2, 3, 4, 80) for n in ("x", "res", "gate"))
    o, s = block_norm_fn(y["x"], y["res"], y["post"], y["pre"], gate=y["gate"], scale=y["scale"], eps=EPS)
    assert o.shape == s.shape == (2, 3, 4, 80)
    compare_border(x, {"out": o.view(24, 80), "s": s.view(24, 80)})


def test_border_weights_of_mixed_types():
    x, up = make_border(6, 48, BF16, BF16, seed=5)
    x["pre"] = x["pre"].float()
    x["scale"] = x["scale"].half()
    got = run_border(x, up)
    assert (got["dpre"].dtype, got["dscale"].dtype, got["dpost"].dtype) == (F32, F16, BF16)
    compare_border(x, got, up)


def test_border_extreme_rows():
    """Zero rows, gates far out, infinities and NaN: each row by itself."""
    x, up = make_border(8, 64, F32, F32, vec=False, seed=6)
    x["x"][0] = 0.0
    x["gate"][1] = 200.0
    x["gate"][2] = -200.0
    want = run_border(x, up)
    compare_border(x, want, up)
    y = dict(x)
    y["x"], y["gate"] = x["x"].clone(), x["gate"].clone()
    y["x"][4, 3], y["x"][5, 7], y["gate"][6, 0] = float("nan"), float("inf"), float("nan")
    got = run_border(y, up)
    keep = [0, 1, 2, 3, 7]
    for n in ("out", "s", "dx", "dres", "dgate"):
        assert torch.equal(got[n][keep], want[n][keep]), n
    assert got["out"][4].isnan().all() and got["out"][6].isnan().all()


def test_border_eps_zero():
    x, up = make_border(5, 33, F32, F32, seed=7)
    o, s = block_norm_fn(x["x"], x["res"], x["post"], x["pre"], gate=x["gate"], scale=x["scale"], eps=0.0)
    want, room = border(**x, eps=0.0)
    check(o, want["out"], room["out"], "out")
    check(s, want["s"], room["s"], "s")


@pytest.mark.parametrize("shape", [(0, 16), (4, 0)], ids=["rows", "dim"])
def test_border_empty(shape):
    x, up = make_border(*shape, F32, F32)
    got = run_border(x, up)
    assert got["out"].shape == shape and got["dpost"].shape == (shape[1],) and not got["dpre"].any()


# ---------------------------------------------------------------- heads --
def make_heads(rows, groups, n, dtype, wtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    D = groups * n
    return {"x": rand(gen, rows, D, dtype=dtype), "gate": rand(gen, rows, D, dtype=dtype, mul=2.0),
            "w": rand(gen, D, dtype=wtype, mul=0.2)}, rand(gen, rows, D, dtype=dtype)


def run_heads(x, groups, dout=None):
    leaves = {n: t.detach().requires_grad_(dout is not None) for n, t in x.items()}
    o = gated_rms_norm_fn(leaves["x"], leaves["gate"], leaves["w"], n_groups=groups, eps=EPS)
    got = {"out": o}
    if dout is not None:
        for n, t in zip(("dx", "dgate", "dweight"), torch.autograd.grad(o, list(leaves.values()), dout)):
            got[n] = t
    return got


def compare_heads(x, groups, got, dout=None):
    want, room = heads(x["x"], x["gate"], x["w"], groups, EPS, dout)
    for n, t in got.items():
        check(t, want[n], room[n], n)


HEADS = [(1, 1, 1), (3, 1, 16), (5, 3, 17), (4, 24, 64), (7, 2, 33), (2, 40, 64), (3, 300, 8), (9, 6, 97), (2, 5, 128), (3, 3, 250),
         (2, 2, 256), (2, 2, 511), (2, 3, 700), (3, 1, 1024), (2, 2, 1500), (2, 1, 4096), (2, 3, 5001), (1, 1, 16384), (130, 1, 30)]


@pytest.mark.parametrize("types", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("shape", HEADS, ids=lambda s: "x".join(map(str, s)))
def test_heads(shape, types):
    x, dout = make_heads(*shape, *types, seed=sum(shape))
    compare_heads(x, shape[1], run_heads(x, shape[1]))
    compare_heads(x, shape[1], run_heads(x, shape[1], dout), dout)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_heads_many_rows(dtype):
    x, dout = make_heads(3000, 3, 40, dtype, dtype, seed=1)
    compare_heads(x, 3, run_heads(x, 3, dout), dout)


def test_heads_layouts():
    x, dout = make_heads(12, 4, 24, BF16, BF16, seed=2)
    wide = torch.zeros(12, 203, dtype=BF16, device=DEV)
    for i, n in enumerate(("x", "gate")):
        wide[:, 3 + 100 * i:99 + 100 * i] = x[n]
        x[n] = wide[:, 3 + 100 * i:99 + 100 * i]
    dout = dout.t().contiguous().t()
    compare_heads(x, 4, run_heads(x, 4, dout), dout)


@pytest.mark.parametrize("shape", [(0, 2, 8), (3, 2, 0)], ids=["rows", "dim"])
def test_heads_empty(shape):
    x, dout = make_heads(*shape, F32, F32)
    got = run_heads(x, shape[1], dout)
    assert got["out"].shape == got["dx"].shape == x["x"].shape and not got["dweight"].any()


def test_refusals():
    t, w = torch.zeros(4, 12, device=DEV), torch.zeros(12, device=DEV)
    for call, msg in ((lambda: block_norm_fn(t, t[:2], w, w), "residual must match"), (lambda: block_norm_fn(t, t, w[:3], w), "post must be"),
                      (lambda: block_norm_fn(t, t, w, w.cpu()), "pre is on"), (lambda: block_norm_fn(t, t.half(), w, w), "residual must match"),
                      (lambda: block_norm_fn(t, t, w, w, gate=t[:, :3]), "gate must match"), (lambda: block_norm_fn(t, t, w, w, eps=-1.0), "eps"),
                      (lambda: block_norm_fn(t, t, w, w, scale=w[:2]), "scale must be"), (lambda: block_norm_fn(t.long(), t.long(), w, w), "dtype"),
                      (lambda: block_norm_fn(t.new_zeros(1, 20000), t.new_zeros(1, 20000), w.new_zeros(20000), w.new_zeros(20000)), "16384"),
                      (lambda: block_norm_fn(t, t, w.long(), w), "float tensor"),
                      (lambda: gated_rms_norm_fn(t, t, w, n_groups=5), "multiple"), (lambda: gated_rms_norm_fn(t, t, w, n_groups=0), "groups"),
                      (lambda: gated_rms_norm_fn(t, t.half(), w), "gate must match"), (lambda: gated_rms_norm_fn(t, t, w[:1]), "weight must be")):
        with pytest.raises(ValueError, match=msg):
            call()


def test_the_same_bits_every_run_and_another_stream():
    x, up = make_border(3000, 768, BF16, F32, seed=8)
    h, dout = make_heads(3000, 12, 64, BF16, F32, seed=9)
    want = [run_border(x, up), run_heads(h, 12, dout)]
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = [run_border(x, up), run_heads(h, 12, dout)]
        torch.cuda.current_stream().wait_stream(side)
        for g, w in zip(got, want):
            for n in w:
                assert torch.equal(g[n], w[n]), n


def test_captured():
    """Both operators and the clipping of their gradients in one graph, replayed on new inputs."""
    def everything(x, up, h, dout):
        b, g = run_border(x, up), run_heads(h, 12, dout)
        grads = [b["dx"], b["dpost"], g["dx"], g["dweight"]]
        clipped = [torch.empty_like(t) for t in grads]
        norm = clip_grads(grads, 1.0, out=clipped)
        return list(b.values()) + list(g.values()) + clipped + [norm]

    def inputs(seed):
        return [*make_border(700, 96, BF16, BF16, seed=seed), *make_heads(500, 12, 64, BF16, BF16, seed=seed)]

    def tensors(i):
        return [*i[0].values(), *i[1].values(), *i[2].values(), i[3]]

    a, b = inputs(10), inputs(11)
    want = [everything(*a), everything(*b)]
    held = inputs(12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = everything(*held)
    for turn in (1, 0, 1):
        for to, t in zip(tensors(held), tensors((a, b)[turn])):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for i, (g, w) in enumerate(zip(got, want[turn])):
            assert torch.equal(g, w), (turn, i)


def test_gradients_against_differences():
    """Directional derivatives against central differences of the kernels' own forward."""
    x, up = make_border(6, 64, F32, F32, seed=13)
    h, dout = make_heads(6, 4, 16, F32, F32, seed=14)
    w = up["dout"].double(), up["ds"].double()

    def border_value(y):
        r = run_border(y)
        return (r["out"].double() * w[0] + r["s"].double() * w[1])

    def heads_value(y):
        return run_heads(y, 4)["out"].double() * dout.double()

    torch.manual_seed(0)
    for value, x0, got in ((border_value, x, run_border(x, up)), (heads_value, h, run_heads(h, 4, dout))):
        names = {"w": "dweight"}
        for n in x0:
            d = torch.randn_like(x0[n])
            step = 2.0 ** -9
            up_, down = (value({**x0, n: x0[n] + s * step * d}) for s in (1, -1))
            slope = float((got[names.get(n, "d" + n)].double() * d.double()).sum())
            # rounding of the two forwards over 2 step, and the third derivative's share (step^2 of order-one terms)
            tol = (64 * 2.0 ** -24 / step + 16 * step * step) * float(up_.abs().sum())
            assert abs(float((up_ - down).sum()) / (2 * step) - slope) <= tol, n


# ------------------------------------------------------------- clipping --
def grads_of(shapes, dtypes, seed=0, mul=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [rand(gen, *s, dtype=t, mul=mul) for s, t in zip(shapes, dtypes)]


def check_clip(before, after, norm, max_norm, eps=1e-6):
    want = math.sqrt(sum(float(g.double().square().sum()) for g in before))
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want, (float(norm), want)
    coef = min(1.0, max_norm / (want + eps))
    for i, (g, o) in enumerate(zip(before, after)):
        # the norm, its sum with eps, the quotient and the product: five roundings
        check(o, g.double().cpu() * coef, 5 * 2.0 ** -24 * g.double().cpu().abs() * coef, f"tensor {i}")


SIZES = [(1,), (0,), (7,), (33, 5), (16384,), (16385,), (100, 331), (2, 3, 4, 5), (70000,)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16, None], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("max_norm", [1.0, 1e6, 0.0])
def test_clip(dtype, max_norm):
    types = [dtype or (F32, BF16, F16)[i % 3] for i in range(len(SIZES))]
    g = grads_of(SIZES, types)
    before = [t.clone() for t in g]
    out = [torch.empty_like(t) for t in g]
    norm = clip_grads(g, max_norm, out=out)
    assert all(torch.equal(a, b) for a, b in zip(g, before))
    check_clip(before, out, norm, max_norm)
    versions = [t._version for t in g]
    again = clip_grads(g, max_norm)
    assert torch.equal(norm, again) and norm.shape == () and norm.dtype == F32
    for a, b, v in zip(g, out, versions):
        assert torch.equal(a, b) and a._version > v


@pytest.mark.parametrize("count", [1, 95, 96, 97, 300])
def test_clip_many_tensors(count):
    g = grads_of([(1 + 37 * (i % 11),) if i % 13 else (0,) for i in range(count)], [F32] * count, seed=count)
    before = [t.clone() for t in g]
    check_clip(before, g, clip_grads(g, 0.5), 0.5)


def test_clip_layouts():
    flat = torch.randn(1000, device=DEV)
    g = [flat[1:301].view(10, 30), torch.randn(20, 30, device=DEV).t(), torch.randn(2, 8, 4, 4, device=DEV).contiguous(memory_format=torch.channels_last),
         flat[501:808].bfloat16()[1:]]
    before = [t.clone() for t in g]
    check_clip(before, g, clip_grads(iter(g + [None]), 1.0), 1.0)


def test_clip_range():
    for mul in (1e-30, 1e30):
        g = grads_of([(300,), (40, 40)], [F32, F32], seed=2, mul=mul)
        before = [t.clone() for t in g]
        check_clip(before, g, clip_grads(g, 1.0, eps=0.0), 1.0, eps=0.0)


def test_clip_not_finite():
    g = grads_of([(300,), (40,)], [F32, BF16], seed=3)
    g[0][5] = float("inf")
    assert float(clip_grads(g, 1.0)) == float("inf")
    assert g[0][5].isnan() and not g[0][:5].any() and not g[1].any()
    g = grads_of([(300,), (40,)], [F32, BF16], seed=3)
    g[1][7] = float("nan")
    assert clip_grads(g, 1.0).isnan() and g[0].isnan().all()


def test_clip_nothing():
    assert float(clip_grads([], 1.0)) == 0.0
    assert float(clip_grads([None, None], 1.0)) == 0.0
    assert float(clip_grads([torch.zeros(0, device=DEV)], 1.0)) == 0.0
    z = [torch.zeros(5, device=DEV)]
    assert float(clip_grads(z, 1.0)) == 0.0 and not z[0].any()


def test_clip_refusals():
    t = torch.zeros(8, 8, device=DEV)
    for call, msg in ((lambda: clip_grads([t[:, ::2]], 1.0), "gaps"), (lambda: clip_grads([t.long()], 1.0), "dtype"),
                      (lambda: clip_grads([t], 1.0, out=[t.half()]), "out must match"), (lambda: clip_grads([t], 1.0, out=[t.t()]), "out must match"),
                      (lambda: clip_grads([t], -1.0), "max_norm"), (lambda: clip_grads([t], float("nan")), "max_norm"),
                      (lambda: clip_grads([t, t.cpu()], 1.0), "one device"), (lambda: clip_grads([t], 1.0, out=[]), "out holds"),
                      (lambda: clip_grads([t[:1].expand(8, 8)], 1.0), "gaps")):
        with pytest.raises(ValueError, match=msg):
            call()
