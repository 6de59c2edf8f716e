"""The delta rule and the norms stay inside their arrays, and depend on nothing that they were not given.

Every input and output, `saved` and the workspaces lie exactly as large as asked for between guards of bytes of ones (NaN
in every type), and outputs, `saved` and workspaces start as such bytes too.  After the calls of the C interface
every guard holds them still, and the results have the bits of the Python calls on tensors of their own.
"""
import pytest
import torch

from mamba_amd import _native as nat
from mamba_amd.ops.delta_rule import delta_rule_fn, delta_rule_update
from mamba_amd.ops.layer_norm import layer_norm_fn
from mamba_amd.ops.unit_norm import unit_norm_fn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
GUARD = 1 << 16
TYPES = {torch.float32: nat.SS_F32, torch.bfloat16: nat.SS_BF16, torch.float16: nat.SS_F16}


class Arena:
    """Tensors between guards."""

    def __init__(self):
        self.all = []

    def room(self, shape, dtype, strides=None):
        """An uninitialised (NaN) tensor; strides in elements."""
        shape = tuple(shape)
        if strides is None:
            strides = [1] * len(shape)
            for i in range(len(shape) - 2, -1, -1):
                strides[i] = strides[i + 1] * max(1, shape[i + 1])
        n = 0 if 0 in shape else 1 + sum((s - 1) * t for s, t in zip(shape, strides))
        size = torch.empty((), dtype=dtype).element_size()
        buf = torch.full((2 * GUARD + (n * size + 255) // 256 * 256,), 255, dtype=torch.uint8, device=DEV)
        view = buf[GUARD:GUARD + n * size].view(dtype).as_strided(shape, strides)
        used = torch.zeros(buf.numel(), dtype=torch.bool, device=DEV)
        for b in range(size if n else 0):
            used[GUARD + b:].as_strided(shape, [s * size for s in strides]).fill_(True)
        self.all.append((buf, used))
        return view

    def put(self, t, strides=None):
        v = self.room(t.shape, t.dtype, strides)
        v.copy_(t)
        return v

    def bytes(self, n):
        return self.room((n,), torch.uint8)

    def check(self):
        for buf, used in self.all:
            assert bool((buf[~used] == 255).all()), "written outside"


def ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def call(name, args):
    import ctypes
    rc = getattr(nat.load(), name)(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, nat.load().ss_last_error()


CASES = [
    # B, L, H, G, K, V, lengths, strided
    (1, 1, 1, 1, 1, 1, None, False), (2, 65, 4, 2, 64, 64, [65, 3], False), (1, 130, 2, 1, 33, 17, None, True),
    (2, 100, 3, 3, 8, 24, [0, 99], True), (1, 1500, 2, 2, 64, 64, None, False), (2, 900, 2, 1, 128, 80, [900, 333], False),
    (1, 300, 1, 1, 256, 256, None, False), (1, 1100, 1, 1, 136, 72, None, True),
]


@pytest.mark.parametrize("dtype", list(TYPES), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])))
@pytest.mark.parametrize("train", [False, True], ids=["prompt", "train"])
def test_delta_rule(case, dtype, train):
    import ctypes
    B, L, H, G, K, V, lengths, strided = case
    gen = torch.Generator().manual_seed(sum(case[:6]))
    x = {n: torch.randn(B, L, h, d, generator=gen).to(dtype).to(DEV) for n, h, d in (("q", G, K), ("k", G, K), ("v", H, V), ("dout", H, V))}
    x["k"] = torch.nn.functional.normalize(x["k"].float(), dim=-1).to(dtype)
    x["g"], x["beta"] = -torch.rand(B, L, H, generator=gen).to(DEV), torch.rand(B, L, H, generator=gen).to(DEV)
    x["initial"], x["dlast"] = (torch.randn(B, H, K, V, generator=gen).to(DEV) for _ in range(2))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    leaves = [x[n].clone().requires_grad_(train) for n in ("q", "k", "v", "g", "beta", "initial")]
    out, last = delta_rule_fn(*leaves[:5], scale=0.5, initial_state=leaves[5], lengths=lens, return_last_state=True)
    want = {"out": out.detach(), "last": last.detach()}
    if train:
        want.update(zip(("dq", "dk", "dv", "dg", "dbeta", "dinitial"), torch.autograd.grad([out, last], leaves, [x["dout"], x["dlast"]])))

    ar = Arena()
    rows = (lambda t: [L * (t.shape[2] * (t.shape[3] + 3) + 5), t.shape[2] * (t.shape[3] + 3) + 5, t.shape[3] + 3, 1]) if strided else lambda t: None
    y = {n: ar.put(t, rows(t) if t.dim() == 4 and n in ("q", "k", "v", "dout") else None) for n, t in x.items()}
    if lens is not None:
        lens = ar.put(lens)
    got = {"out": ar.room((B, L, H, V), dtype, rows(x["v"])), "last": ar.room((B, H, K, V), torch.float32)}
    a = nat.DeltaRuleArgs(batch=B, seqlen=L, heads=H, groups=G, d_key=K, d_value=V, dtype=TYPES[dtype], scale=0.5)

    def strides(args, n, t):
        for i, d in enumerate(("batch", "len", "head")):
            setattr(args, f"{n}_{d}_stride", t.stride(i))
    for n in ("q", "k", "v", "g", "beta"):
        strides(a, n, y[n])
        setattr(a, n, ptr(y[n]))
    strides(a, "out", got["out"])
    a.initial_state, a.lengths, a.out, a.last_state = ptr(y["initial"]), ptr(lens), ptr(got["out"]), ptr(got["last"])
    if train:
        a.saved_bytes = nat.load().ss_delta_rule_saved_bytes(ctypes.byref(a))
        saved = ar.bytes(a.saved_bytes)
        a.saved = ptr(saved)
    a.workspace_bytes = nat.load().ss_delta_rule_fwd_workspace_bytes(ctypes.byref(a))
    ws = ar.bytes(a.workspace_bytes)
    a.workspace = ptr(ws)
    call("ss_delta_rule_fwd", a)
    if train:
        for n, t in (("dq", x["q"]), ("dk", x["k"]), ("dv", x["v"]), ("dg", x["g"]), ("dbeta", x["beta"]), ("dinitial", x["initial"])):
            got[n] = ar.room(t.shape, t.dtype)
        b = nat.DeltaRuleBwdArgs(f=a)
        strides(b, "dout", y["dout"])
        b.dout, b.dlast_state = ptr(y["dout"]), ptr(y["dlast"])
        b.dq, b.dk, b.dv, b.dg, b.dbeta, b.dinitial_state = (ptr(got[n]) for n in ("dq", "dk", "dv", "dg", "dbeta", "dinitial"))
        b.f.workspace, b.f.workspace_bytes = None, 0
        n = nat.load().ss_delta_rule_bwd_workspace_bytes(ctypes.byref(b))
        ws2 = ar.bytes(n)
        b.f.workspace, b.f.workspace_bytes = ptr(ws2), n
        call("ss_delta_rule_bwd", b)
    ar.check()
    for n, t in got.items():
        assert same(t, want[n]), n


@pytest.mark.parametrize("dtype", list(TYPES), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 1), (3, 2, 1, 33, 17), (2, 4, 4, 64, 64), (2, 2, 1, 200, 256)], ids=lambda c: "x".join(map(str, c)))
def test_update(case, dtype):
    B, H, G, K, V = case
    gen = torch.Generator().manual_seed(sum(case))
    q, k, v = (torch.randn(B, h, d, generator=gen).to(dtype).to(DEV) for h, d in ((G, K), (G, K), (H, V)))
    g, beta = -torch.rand(B, H, generator=gen).to(DEV), torch.rand(B, H, generator=gen).to(DEV)
    state = torch.randn(B, H, K, V, generator=gen).to(DEV)
    ar = Arena()
    s2, out = ar.put(state, [H * (K * V + 8), K * V + 8, V, 1]), ar.room((B, H, V), dtype, [H * (V + 1), V + 1, 1])
    delta_rule_update(s2, ar.put(q), ar.put(k), ar.put(v), ar.put(g), ar.put(beta), scale=0.5, out=out)
    want = delta_rule_update(state, q, k, v, g, beta, scale=0.5)
    ar.check()
    assert same(s2, state) and same(out, want)


@pytest.mark.parametrize("dtype", list(TYPES), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 17), (65, 768), (7, 1001), (5, 4100), (2, 16384)])
def test_norms(rows, dim, dtype):
    import ctypes
    gen = torch.Generator().manual_seed(rows + dim)
    x, r, do, ds = (torch.randn(rows, dim, generator=gen).to(dtype).to(DEV) for _ in range(4))
    w, b = (torch.randn(dim, generator=gen).to(dtype).to(DEV) for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    out, s = layer_norm_fn(leaves[0], leaves[1], leaves[2], residual=leaves[3], prenorm=True)
    grads = torch.autograd.grad([out, s], leaves, [do, ds])
    ar = Arena()
    wide = [dim + 3, 1]
    y = {n: ar.put(t, wide) for n, t in (("x", x), ("r", r), ("do", do), ("ds", ds))}
    y.update(w=ar.put(w), b=ar.put(b), out=ar.room((rows, dim), dtype, wide), s=ar.room((rows, dim), dtype, wide), stats=ar.room((rows, 2), torch.float32))
    a = nat.LayerNormArgs(rows=rows, dim=dim, dtype=TYPES[dtype], w_dtype=TYPES[dtype], eps=1e-5, x_row_stride=dim + 3, residual_row_stride=dim + 3,
                          out_row_stride=dim + 3, residual_out_row_stride=dim + 3, x=ptr(y["x"]), residual=ptr(y["r"]), weight=ptr(y["w"]),
                          bias=ptr(y["b"]), out=ptr(y["out"]), residual_out=ptr(y["s"]), stats=ptr(y["stats"]))
    call("ss_layer_norm_fwd", a)
    n = nat.load().ss_layer_norm_bwd_workspace_bytes(rows, dim)
    ws, dx, dw, db = ar.bytes(n), ar.room((rows, dim), dtype), ar.room((dim,), dtype), ar.room((dim,), dtype)
    g = nat.LayerNormBwdArgs(rows=rows, dim=dim, dtype=TYPES[dtype], w_dtype=TYPES[dtype], s_row_stride=dim + 3, dout_row_stride=dim + 3,
                             dresidual_out_row_stride=dim + 3, s=ptr(y["s"]), weight=ptr(y["w"]), stats=ptr(y["stats"]), dout=ptr(y["do"]),
                             dresidual_out=ptr(y["ds"]), dx=ptr(dx), dweight=ptr(dw), dbias=ptr(db), workspace=ptr(ws), workspace_bytes=n)
    call("ss_layer_norm_bwd", g)
    ux = ar.put(x, wide)
    uo = unit_norm_fn(ux)
    ar.check()
    for got, want in ((y["out"], out), (y["s"], s), (dx, grads[0]), (dw, grads[1]), (db, grads[2]), (dx, grads[3]), (uo, unit_norm_fn(x))):
        assert same(got, want.detach())
