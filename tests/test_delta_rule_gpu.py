"""delta_rule_fn and delta_rule_update on the GPU against the float64 recurrence,
within bounds that tests/_delta_rule_ref.py derives."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from mamba_amd.ops.delta_rule import delta_rule_fn, delta_rule_update
from tests._delta_rule_ref import bounds, check, recurrence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])


def make(B, L, H, G, K, V, dtype, seed=0, initial=False, lengths=None, decay=0.2):
    gen = torch.Generator().manual_seed(seed)
    x = {n: torch.randn(B, L, h, d, generator=gen) for n, h, d in (("q", G, K), ("k", G, K), ("v", H, V), ("dout", H, V))}
    x["k"] = x["k"] / torch.linalg.vector_norm(x["k"], dim=-1, keepdim=True)
    x = {n: t.to(dtype) for n, t in x.items()}
    x["g"] = -torch.rand(B, L, H, generator=gen) * decay
    x["beta"] = torch.sigmoid(torch.randn(B, L, H, generator=gen))
    x["initial"] = torch.randn(B, H, K, V, generator=gen) if initial else None
    x["dlast"] = torch.randn(B, H, K, V, generator=gen) if initial else None
    x["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return {n: None if t is None else t.to(DEV) for n, t in x.items()}


def run(x, grad=True, scale=None):
    leaves = {n: x[n].detach().requires_grad_(grad) for n in ("q", "k", "v", "g", "beta", "initial") if x[n] is not None}
    o, last = delta_rule_fn(leaves["q"], leaves["k"], leaves["v"], leaves["g"], leaves["beta"], scale=scale,
                            initial_state=leaves.get("initial"), lengths=x["lengths"], return_last_state=True)
    got = {"out": o, "last": last}
    if grad:
        outs, ups = ([o, last], [x["dout"], x["dlast"]]) if x["dlast"] is not None else ([o], [x["dout"]])
        for n, t in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups)):
            got["d" + n] = t
    return got


def compare(x, got, scale=None):
    s = x["q"].shape[-1] ** -0.5 if scale is None else scale
    grads = (x["dout"], x["dlast"]) if "dq" in got else ()
    want = recurrence(x["q"], x["k"], x["v"], x["g"], x["beta"], s, x["initial"], x["lengths"], *grads)
    room = bounds(want, x["v"].dtype, abs(s))
    for n, t in got.items():
        check(t, want[n], room[n], n)
    return want


SHAPES = [
    # B, L, H, G, K, V
    (1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 16, 16), (1, 3, 2, 2, 7, 5), (2, 63, 2, 2, 64, 64), (1, 64, 3, 1, 64, 64),
    (2, 65, 2, 2, 64, 64), (1, 127, 4, 2, 32, 128), (1, 200, 2, 1, 128, 64), (2, 130, 2, 2, 96, 80), (1, 513, 2, 2, 20, 24),
    (1, 1030, 2, 2, 64, 64), (1, 150, 1, 1, 130, 200), (1, 140, 1, 1, 256, 256), (3, 90, 6, 2, 48, 33), (1, 2100, 1, 1, 16, 65),
    (1, 1100, 1, 1, 160, 16),
]


@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(shape, dtype):
    x = make(*shape, dtype, seed=sum(shape), initial=shape[1] % 2 == 1)
    compare(x, run(x))


WHOLE = [
    # rows of whole 16-byte vectors, narrower than the tiles
    (1, 70, 2, 2, 8, 8), (2, 65, 3, 1, 24, 16), (1, 100, 2, 1, 72, 40), (1, 129, 2, 2, 136, 24), (1, 97, 1, 1, 200, 136),
    # many segments, at every tile of keys
    (1, 4000, 1, 1, 64, 64), (1, 1700, 2, 1, 128, 128), (1, 1500, 1, 1, 256, 48),
]


@TYPES
@pytest.mark.parametrize("shape", WHOLE, ids=lambda s: "x".join(map(str, s)))
def test_whole_rows_and_segments(shape, dtype):
    x = make(*shape, dtype, seed=50 + sum(shape), initial=True)
    compare(x, run(x))


@TYPES
def test_lengths_within_segments(dtype):
    """Rows that end in the first, a middle and the last segment, and one without tokens."""
    lengths = [0, 100, 1000, 1699, 1700]
    x = make(5, 1700, 1, 1, 96, 64, dtype, seed=51, initial=True, lengths=lengths)
    got = run(x)
    compare(x, got)
    for b, n in enumerate(lengths):
        for name in ("out", "dq", "dk", "dv", "dg", "dbeta"):
            assert not got[name][b, n:].any(), (name, n)


def test_lengths_of_64_bits():
    """Whole numbers of either width, past 32 bits too."""
    x = make(4, 100, 2, 2, 32, 32, F32, seed=53, initial=True, lengths=[0, 37, 100, 100])
    want = run(x)
    x["lengths"] = torch.tensor([-(1 << 40), 37, 1 << 32, (1 << 40) + 5], device=DEV)
    got = run(x)
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_backward_twice():
    """What a forward keeps is left as it is by a backward."""
    for L in (200, 2000):
        x = make(1, L, 2, 1, 64, 64, BF16, seed=52, initial=True)
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "beta", "initial")]
        o, last = delta_rule_fn(*leaves[:5], initial_state=leaves[5], return_last_state=True)
        first = torch.autograd.grad([o, last], leaves, [x["dout"], x["dlast"]], retain_graph=True)
        torch.autograd.grad([o], leaves, [x["dout"] * 2], retain_graph=True)
        for a, b in zip(first, torch.autograd.grad([o, last], leaves, [x["dout"], x["dlast"]])):
            assert torch.equal(a, b)


@TYPES
@pytest.mark.parametrize("shape", [(2, 1100, 4, 4, 64, 64), (1, 700, 2, 2, 128, 128)], ids=lambda s: "x".join(map(str, s)))
def test_precision(shape, dtype):
    """Rms errors.  A result is a sum whose terms carry some tens of roundings of 2^-25 rms, of either sign, on
    the way: fp32 ones stay within 2^-20 of their rms (dg, whose terms cancel, 2^-19); two 16-bit terms in a
    state's or a 32-bit gradient's way (2^-17 and more) do not.  16-bit results: their own rounding, 0.29 of a step rms,
    at most 0.42 eps beside it."""
    x = make(*shape, dtype, seed=40, initial=True)
    got, want = run(x), recurrence(*(x[n] for n in ("q", "k", "v", "g", "beta")), x["q"].shape[-1] ** -0.5, x["initial"], None, x["dout"], x["dlast"])
    for n, t in got.items():
        e = float((t.double().cpu() - want[n]).square().mean().sqrt() / want[n].square().mean().sqrt())
        room = 0.42 * torch.finfo(t.dtype).eps if t.dtype != F32 else 2.0 ** -19 if n == "dg" else 2.0 ** -20
        assert e <= room, (n, e)


def test_many_rows():
    """More rows than compute units, of all lengths."""
    x = make(600, 140, 2, 1, 16, 16, BF16, seed=30, initial=True, lengths=[(7 * i) % 141 for i in range(600)])
    compare(x, run(x))


@TYPES
@pytest.mark.parametrize("L", [150, 1300])
def test_lengths(dtype, L):
    """What lies past a row's length is not read; whole segments past it too."""
    lengths = [0, 1, 64, 65, L, L - 1] if L == 150 else [0, 700]
    x = make(len(lengths), L, 4 if L == 150 else 2, 2, 64, 64, dtype, seed=4, initial=True, lengths=lengths)
    for b, n in enumerate(lengths):
        for t in ("q", "k", "v", "dout"):
            x[t][b, n:] = float("nan")
        x["g"][b, n:] = float("inf")
        x["beta"][b, n:] = float("nan")
    got = run(x)
    y = dict(x)
    for b, n in enumerate(lengths):
        for t in ("q", "k", "v", "dout", "g", "beta"):
            y[t] = y[t].clone() if y[t] is x[t] else y[t]
            y[t][b, n:] = 0.0
    compare(y, got)
    assert torch.equal(got["last"][0], x["initial"][0])


def test_lengths_beyond_the_row():
    x = make(2, 70, 2, 2, 32, 32, F32, seed=5, lengths=[1000, -3])
    compare(x, run(x))


@TYPES
def test_decays_at_their_ends(dtype):
    """Resets (minus infinity, the type's lowest value), no decay."""
    x = make(2, 200, 4, 4, 64, 64, dtype, seed=6, initial=True)
    lowest = torch.finfo(F32).min
    for b, t, h, v in ((0, 0, 0, -float("inf")), (0, 100, 0, -float("inf")), (0, 101, 0, lowest), (1, 63, 1, lowest),
                       (1, 64, 1, -float("inf")), (0, 199, 2, -float("inf")), (1, 10, 3, -90.0), (1, 130, 3, -200.0)):
        x["g"][b, t, h] = v
    x["g"][0, :, 3] = 0.0
    got = run(x)
    compare(x, got)
    assert not got["dg"][x["g"] < -150].any()


def test_strong_decays_gradient():
    """dg of a token has the factor exp(g): relative to it, its error is that of any other token's."""
    x = make(1, 300, 2, 2, 64, 64, F32, seed=7, initial=True)
    at = torch.arange(20, 300, 37)
    x["g"][0, at, :] = -torch.linspace(5.0, 60.0, len(at), device=DEV)[:, None]
    got, want = run(x), recurrence(*(x[n] for n in ("q", "k", "v", "g", "beta")), 0.125, x["initial"], None, x["dout"], x["dlast"])
    room = bounds(want, F32, 0.125)["dg"]
    factor = torch.exp(x["g"].double().cpu())
    check((got["dg"].double().cpu() / factor)[0, at].float(), (want["dg"] / factor)[0, at], room[0, at] + 2.0 ** -22 * (want["dg"] / factor)[0, at].abs(), "dg")


@TYPES
def test_rates_at_their_ends(dtype):
    """beta of 0 (nothing is written), 1 (what the key held is replaced), 2 (reflected), tiny and negative ones."""
    x = make(1, 200, 4, 4, 64, 64, dtype, seed=8, initial=True)
    x["beta"][0, ::3, 0] = 0.0
    x["beta"][0, :, 1] = 1.0
    x["beta"][0, ::2, 2] = 2.0 - 2.0 ** -6                     # (a rounded key is up to 2^-8 longer than one)
    x["beta"][0, 5::7, 3], x["beta"][0, 6::7, 3], x["beta"][0, 7::7, 3] = 1e-30, -0.0, 1e-42
    got = run(x)
    compare(x, got)
    assert not got["dv"][0, ::3, 0].any()


def test_nothing_is_written():
    """beta of 0 throughout: the state only decays, and dbeta still says what a rate would change."""
    x = make(1, 150, 1, 1, 32, 32, F32, seed=9, initial=True)
    x["beta"].zero_()
    x["g"].zero_()
    got = run(x)
    compare(x, got)
    assert torch.equal(got["last"], x["initial"]) and got["dbeta"].abs().min() > 0


@TYPES
def test_equal_keys(dtype):
    """One key throughout: the triangular system that powers of its matrix do not solve in 32 bits."""
    x = make(1, 200, 2, 2, 64, 64, dtype, seed=10, initial=True)
    x["k"] = x["k"][:, :1].expand_as(x["k"]).contiguous()
    x["g"].zero_()
    x["beta"][..., 0], x["beta"][..., 1] = 1.0, 1.9
    compare(x, run(x))


def test_longer_keys():
    """Keys longer than one, with rates that keep them contracting."""
    x = make(2, 200, 2, 1, 64, 64, F32, seed=11, initial=True)
    x["k"], x["beta"] = x["k"] * 8, x["beta"] / 64
    compare(x, run(x))


def test_another_token_stays_in_its_row():
    """Infinities and NaN of a token leave other rows and heads, and the chunks before its own, alone."""
    for dtype in (F32, BF16, F16):
        x = make(2, 150, 2, 2, 64, 64, dtype, seed=12)
        want = run(x, grad=False)["out"]
        for n, v in (("v", float("nan")), ("k", float("inf")), ("q", float("nan"))):
            y = dict(x)
            y[n] = x[n].clone()
            y[n][0, 130, 0, 3] = v
            got = run(y, grad=False)["out"]
            assert torch.equal(got[1], want[1]) and torch.equal(got[0, :, 1], want[0, :, 1]) and torch.equal(got[0, :128, 0], want[0, :128, 0])
            assert not got[0, 130, 0].isfinite().all()


LAYOUTS = {
    "one projection": None,
    "heads first": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
    "rows off 16 bytes": lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2],
    "every second column": lambda t: t.repeat_interleave(2, -1)[..., ::2],
    "batch broadcast": lambda t: t[:1].expand_as(t),
}


@TYPES
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_layouts(layout, dtype):
    x = make(2, 140, 4, 2, 64, 48, dtype, seed=13)
    if layout == "one projection":
        row = torch.cat([x[n].flatten(2) for n in ("q", "k", "v")], -1)
        q, k, v = row.split([128, 128, 192], -1)
        x["q"], x["k"], x["v"] = q.view(2, 140, 2, 64), k.view(2, 140, 2, 64), v.view(2, 140, 4, 48)
        x["g"], x["beta"] = x["g"][:, :, :1].expand(2, 140, 4), x["beta"][:1, :1].expand(2, 140, 4)
    else:
        for n in ("q", "k", "v", "dout"):
            x[n] = LAYOUTS[layout](x[n])
        x["g"], x["beta"] = (x[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("g", "beta"))
    compare(x, run(x))


def test_factors_in_the_rows_type():
    x = make(2, 100, 2, 2, 32, 32, BF16, seed=14)
    x["g"], x["beta"] = x["g"].bfloat16(), x["beta"].bfloat16()
    got = run(x)
    assert got["dg"].dtype == got["dbeta"].dtype == BF16
    compare(x, got)


def test_only_some_gradients():
    x = make(1, 80, 2, 2, 32, 32, F32, seed=15, initial=True)
    v = x["v"].detach().requires_grad_()
    o = delta_rule_fn(x["q"], x["k"], v, x["g"], x["beta"], initial_state=x["initial"])
    alone, = torch.autograd.grad(o, [v], x["dout"])
    x["dlast"] = torch.zeros_like(x["dlast"])
    full = run(x)
    assert torch.equal(alone, full["dv"]) and torch.equal(o.detach(), full["out"].detach())
    i = x["initial"].detach().requires_grad_()
    _, last = delta_rule_fn(x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=i, return_last_state=True)
    di, = torch.autograd.grad(last.sum(), [i])
    x["dout"], x["dlast"] = torch.zeros_like(x["dout"]), torch.ones_like(x["dlast"])
    compare(x, {"dinitial": di, "dq": torch.zeros_like(x["q"])})


@pytest.mark.parametrize("shape", [(0, 5, 2, 2, 8, 8), (2, 0, 2, 1, 8, 8), (2, 5, 0, 1, 8, 8)], ids=["batch", "seqlen", "heads"])
def test_empty(shape):
    x = make(*shape, F32, initial=True)
    got = run(x)
    assert got["out"].shape == x["v"].shape and got["dq"].shape == x["q"].shape and not got["dq"].any()
    assert torch.equal(got["last"], x["initial"]) and torch.equal(got["dinitial"], x["dlast"])
    assert got["dg"].shape == got["dbeta"].shape == x["g"].shape


def test_gradient_against_differences():
    """The derivative along a direction against central differences of the forward."""
    x = make(1, 130, 2, 1, 32, 32, F32, seed=16, initial=True)
    got = run(x)
    torch.manual_seed(0)
    w = x["dout"].double(), x["dlast"].double()

    def value(y):
        r = run(y, grad=False)
        return float((r["out"].double() * w[0]).sum() + (r["last"].double() * w[1]).sum())

    def exact(y):                     # the same difference of the float64 recurrence: its third derivative's share
        r = recurrence(*(y[n] for n in ("q", "k", "v", "g", "beta")), 32 ** -0.5, y["initial"])
        return float((r["out"] * w[0].cpu()).sum() + (r["last"] * w[1].cpu()).sum())

    for n in ("q", "k", "v", "g", "beta", "initial"):
        d = torch.randn_like(x[n]) * (0.05 if n in ("g", "beta", "k") else 1.0)
        h = 2.0 ** -7
        ends = [{**x, n: x[n] + s * h * d} for s in (1, -1)]
        up, down = map(value, ends)
        slope = float((got["d" + n].double() * d.double()).sum())
        third = abs((exact(ends[0]) - exact(ends[1])) / (2 * h) - float((recurrence(*(x[m] for m in ("q", "k", "v", "g", "beta")), 32 ** -0.5,
                    x["initial"], None, x["dout"], x["dlast"])["d" + n] * d.double().cpu()).sum()))
        # the forward's rounding over 2 h
        tol = 2.0 ** -16 * abs(slope) + third * 1.01 + 2.0 ** -20 / h * float((got["out"].double() * w[0]).abs().sum() + (got["last"].double() * w[1]).abs().sum())
        assert abs((up - down) / (2 * h) - slope) <= tol, n


def test_the_same_bits_every_run():
    x = make(2, 700, 4, 2, 64, 64, BF16, seed=17, initial=True)
    a, b = run(x), run(x)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_another_stream():
    x = make(1, 1500, 2, 2, 64, 64, BF16, seed=18)
    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("L", [300, 1500])
def test_captured(L):
    """Forward and backward in one graph, replayed on new inputs with eager work between."""
    x = make(2, L, 2, 1, 64, 64, BF16, seed=19, initial=True)
    y = make(2, L, 2, 1, 64, 64, BF16, seed=20, initial=True)
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
        again = run((x, y)[1 - turn])
        for n in got:
            assert torch.equal(got[n], want[turn][n]) and torch.equal(again[n], want[1 - turn][n]), (turn, n)


def test_far_rows():
    """Row offsets past 2^31 elements."""
    far = torch.zeros((1 << 31) + 70 * 64 + 64, dtype=BF16, device=DEV)
    x = make(2, 70, 1, 1, 64, 64, BF16, seed=21)
    want = run(x)
    for n in ("q", "k", "v", "dout"):
        y = dict(x)
        y[n] = far.as_strided((2, 70, 1, 64), (1 << 31, 64, 64, 1))
        y[n].copy_(x[n])
        got = run(y)
        for m in want:
            assert torch.equal(got[m], want[m]), (n, m)


def test_derivatives_it_does_not_have():
    x = make(1, 40, 2, 2, 16, 8, F32, seed=22, initial=True)
    names = ("q", "k", "v", "g", "beta", "initial")

    def call(y):
        return delta_rule_fn(y["q"], y["k"], y["v"], y["g"], y["beta"], initial_state=y["initial"])

    for n in names:
        with fwad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            call({**x, n: fwad.make_dual(x[n], torch.ones_like(x[n]))})
        y = {**x, n: x[n].clone().requires_grad_()}
        first, = torch.autograd.grad(call(y).sum(), [y[n]])
        graph, = torch.autograd.grad(call(y).sum(), [y[n]], create_graph=True)
        assert torch.equal(first, graph)
        with pytest.raises(RuntimeError, match="second"):
            (graph.square().sum() + y[n].square().sum()).backward()
        y[n].grad = None


# ------------------------------------------------------------ one token --
def _token(B, H, G, K, V, dtype, seed=0):
    x = make(B, 1, H, G, K, V, dtype, seed=seed, initial=True)
    return x, [x[n][:, 0] for n in ("q", "k", "v", "g", "beta")]


@TYPES
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 24, 24, 64, 64), (64, 4, 2, 128, 128), (3, 6, 2, 96, 80), (2, 2, 1, 7, 33),
                                   (5, 2, 2, 256, 256), (2, 3, 3, 130, 6), (2, 1, 1, 200, 100)], ids=lambda s: "x".join(map(str, s)))
def test_update(shape, dtype):
    x, t = _token(*shape, dtype, seed=sum(shape))
    state = x["initial"].clone()
    o = delta_rule_update(state, *t)
    compare(x, {"out": o[:, None], "last": state})


def test_update_continues_the_prompt():
    x = make(2, 100, 4, 2, 64, 64, BF16, seed=23)
    want, whole = delta_rule_fn(*(x[n] for n in ("q", "k", "v", "g", "beta")), return_last_state=True)
    _, state = delta_rule_fn(*(x[n][:, :90] for n in ("q", "k", "v", "g", "beta")), return_last_state=True)
    out = torch.empty_like(x["v"][:, 0])
    for t in range(90, 100):
        r = delta_rule_update(state, *(x[n][:, t] for n in ("q", "k", "v", "g", "beta")), out=out)
        assert r is out
        # both sides within the bounds of the recurrence: twice half a step of the larger plus the sums'
        assert (r.double() - want[:, t].double()).abs().max() <= 2.0 ** -7 * want[:, t].double().abs().max()
    assert (state - whole).abs().max() <= 2.0 ** -14 * whole.abs().max()


def test_update_resets_and_strides():
    x, t = _token(2, 4, 2, 64, 64, F32, seed=24)
    big = torch.zeros(2, 8, 64, 64, device=DEV)
    state = big[:, ::2]
    state.copy_(x["initial"])
    t[3], t[4] = t[3].clone(), t[4].clone()
    t[3][0, 1], t[3][1, 2], t[4][1, 3] = -float("inf"), torch.finfo(F32).min, 0.0
    x["g"], x["beta"] = t[3][:, None], t[4][:, None]
    o = delta_rule_update(state, *t)
    compare(x, {"out": o[:, None], "last": state})
    assert not big[:, 1::2].any()
    off = torch.zeros(2 * 4 * 64 * 64 + 1, device=DEV)[1:].view(2, 4, 64, 64)   # rows off 16 bytes
    off.copy_(x["initial"])
    o2 = delta_rule_update(off, *t)
    compare(x, {"out": o2[:, None], "last": off})


def test_update_captured():
    x, t = _token(2, 4, 4, 64, 64, BF16, seed=25)
    state = x["initial"].clone()
    delta_rule_update(state, *t)
    want = state.clone()
    state.copy_(x["initial"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        delta_rule_update(state, *t)
    for _ in range(3):
        state.copy_(x["initial"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(state, want)


def test_update_refusals():
    x, t = _token(2, 4, 2, 32, 24, F32, seed=26)
    state = x["initial"]
    before = state.clone()
    for i in range(5):
        y = list(t)
        y[i] = y[i].clone().requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            delta_rule_update(state, *y)
        with fwad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            y[i] = fwad.make_dual(t[i], t[i])
            delta_rule_update(state, *y)
    for bad in (state[:1].expand_as(state), state[:, :1].expand_as(state)):
        with pytest.raises(ValueError, match="state's elements overlap"):
            delta_rule_update(bad, *t)
    with pytest.raises(ValueError, match="out's elements overlap"):
        delta_rule_update(state, *t, out=torch.empty_like(t[2][:1]).expand(2, 4, 24))
    with pytest.raises(ValueError, match="contiguous along its last two"):
        delta_rule_update(state.transpose(2, 3).contiguous().transpose(2, 3), *t)
    with pytest.raises(ValueError, match="beta has shape"):
        delta_rule_update(state, *t[:4], t[4][:, :2])
    with pytest.raises(ValueError, match="k has dtype"):
        delta_rule_update(state, t[0], t[1].bfloat16(), *t[2:])
    assert torch.equal(state, before)
    q = x["q"].clone().requires_grad_()
    out = delta_rule_fn(q, x["k"], x["v"], x["g"], x["beta"], initial_state=state)
    version = state._version
    delta_rule_update(state, *t)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals():
    x = make(2, 10, 4, 2, 16, 16, F32, seed=27, initial=True)
    a = [x[n] for n in ("q", "k", "v", "g", "beta")]
    for i, bad, msg in ((0, x["q"][..., :8], "k has shape"), (1, x["k"].half(), "k has dtype"), (2, x["v"][:, :, :3], "multiple of groups"),
                        (3, x["g"][:, :9], "g has shape"), (4, x["beta"].double(), "beta has dtype"), (3, x["g"].cpu(), "g is on"),
                        (2, x["v"][0], "v must be")):
        y = list(a)
        y[i] = bad
        with pytest.raises(ValueError, match=msg):
            delta_rule_fn(*y)
    with pytest.raises(ValueError, match="initial_state has shape"):
        delta_rule_fn(*a, initial_state=x["initial"][:1])
    with pytest.raises(ValueError, match="lengths must be"):
        delta_rule_fn(*a, lengths=torch.ones(2, device=DEV))
    with pytest.raises(ValueError, match="d_key"):
        w = torch.zeros(2, 10, 2, 257, device=DEV)
        delta_rule_fn(w, w, *a[2:])
