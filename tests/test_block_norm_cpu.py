"""Refusals of the norms around a block and of gradient clipping: argument
blocks through the C ABI and tensors through Python, no device work; and the
float64 closed forms against differences."""
import ctypes
import os
import subprocess

import pytest
import torch

from mamba_amd import _native as nat
from mamba_amd.ops.block_norm import block_norm_fn, gated_rms_norm_fn
from mamba_amd.ops.clip_grads import clip_grads
from tests._block_norm_ref import border, heads

FAKE = 1 << 20   # aligned, never dereferenced


def fill(a, names):
    for i, n in enumerate(names):
        setattr(a, n, FAKE + 65536 * i)
    return a


def border_block(bwd):
    a = nat.BlockNormBwdArgs() if bwd else nat.BlockNormArgs()
    a.rows, a.dim, a.dtype, a.w_dtype = 8, 64, nat.SS_BF16, nat.SS_F32
    names = ["x", "residual", "gate", "post", "pre", "scale_vec", "rstd"]
    names += ["dout", "dresidual_out", "dx", "dresidual", "dgate", "dpost", "dpre", "dscale", "workspace"] if bwd else ["out", "residual_out"]
    for n in ("x", "residual", "gate"):
        setattr(a, n + "_row_stride", 64)
    if bwd:
        a.workspace_bytes = 1 << 20
    else:
        a.eps = 1e-6
    return fill(a, names)


def heads_block(bwd):
    a = nat.GatedNormBwdArgs() if bwd else nat.GatedNormArgs()
    a.rows, a.dim, a.groups, a.dtype, a.w_dtype, a.eps = 8, 64, 4, nat.SS_F16, nat.SS_F16, 1e-6
    if bwd:
        a.workspace_bytes = 1 << 20
    return fill(a, ["x", "gate", "weight"] + (["dout", "dx", "dgate", "dweight", "workspace"] if bwd else ["out"]))


COMMON = [("rows", -1, "INVALID", "negative size"), ("dtype", 7, "INVALID", "dtype"), ("w_dtype", 9, "UNSUPPORTED", "weight dtype"),
          ("dim", 16385, "UNSUPPORTED", "above 16384"), ("x", None, "INVALID", "x is NULL"), ("gate", FAKE + 1, "INVALID", "misaligned"),
          ("x_row_stride", -4, "INVALID", "stride")]
BORDER = [("residual", None, "INVALID", "residual is NULL"), ("post", None, "INVALID", "post is NULL"), ("pre", FAKE + 2, "INVALID", "misaligned")]
FWD = [("eps", -1.0, "INVALID", "eps"), ("eps", float("nan"), "INVALID", "eps"), ("out", None, "INVALID", "out is NULL")]
BWD = [("dx", None, "INVALID", "dx is NULL"), ("dgate", None, "INVALID", "dgate is NULL"), ("workspace", None, "INVALID", "workspace"),
       ("workspace_bytes", 4, "INVALID", "workspace"), ("workspace", FAKE + 8, "INVALID", "aligned")]


@pytest.mark.parametrize("kind", ["border", "heads"])
@pytest.mark.parametrize("bwd", [False, True], ids=["fwd", "bwd"])
def test_norm_blocks_refused(kind, bwd):
    lib = nat.load()
    make = border_block if kind == "border" else heads_block
    fn = getattr(lib, f"ss_{'block' if kind == 'border' else 'gated'}_norm_{'bwd' if bwd else 'fwd'}")
    extra = BORDER + ([("rstd", None, "INVALID", "rstd is NULL"), ("dpre", None, "INVALID", "dpre")] if bwd else
                      [("residual_out", None, "INVALID", "residual_out is NULL")]) if kind == "border" else \
        [("groups", 0, "INVALID", "groups"), ("groups", 7, "INVALID", "multiple"), ("weight", None, "INVALID", "weight is NULL")] + \
        ([("dout", None, "INVALID", "dout is NULL"), ("eps", -1.0, "INVALID", "eps")] if bwd else [])
    for field, value, code, msg in COMMON + extra + (BWD if bwd else FWD):
        a = make(bwd)
        setattr(a, field, value)
        assert fn(ctypes.byref(a), None) == getattr(nat, f"SS_ERR_{code}"), field
        assert msg in lib.ss_last_error().decode(), (field, lib.ss_last_error())
    assert fn(None, None) == nat.SS_ERR_INVALID


def test_workspace_sizes():
    lib = nat.load()
    assert lib.ss_block_norm_bwd_workspace_bytes(0, 64) == 0
    assert lib.ss_block_norm_bwd_workspace_bytes(1 << 40, 64) > 0
    assert lib.ss_block_norm_bwd_workspace_bytes(-1, 64) == -1 and lib.ss_block_norm_bwd_workspace_bytes(4, 1 << 20) == -1
    assert lib.ss_gated_norm_bwd_workspace_bytes(9, 64, 4) > 0 and lib.ss_gated_norm_bwd_workspace_bytes(0, 64, 4) == 0
    assert lib.ss_gated_norm_bwd_workspace_bytes(9, 64, 5) == -1 and lib.ss_gated_norm_bwd_workspace_bytes(9, 64, 0) == -1


def clip_block(n=2):
    a = nat.ClipGradsArgs()
    a.count, a.max_norm, a.eps, a.norm, a.workspace, a.workspace_bytes = n, 1.0, 1e-6, FAKE, FAKE, 1 << 20
    keep = ((ctypes.c_void_p * n)(*([FAKE] * n)), (ctypes.c_void_p * n)(*([FAKE] * n)), (ctypes.c_int64 * n)(*([100] * n)),
            (ctypes.c_int32 * n)(*([nat.SS_BF16] * n)))
    a.grads, a.outs, a.numels, a.dtypes = (ctypes.cast(k, ctypes.c_void_p) for k in keep)
    return a, keep


def test_clip_blocks_refused():
    lib = nat.load()

    def refused(a, code, msg):
        assert lib.ss_clip_grads(ctypes.byref(a), None) == code and msg in lib.ss_last_error().decode(), lib.ss_last_error()

    for field, value, msg in (("count", -1, "negative count"), ("grads", None, "NULL"), ("numels", None, "NULL"), ("max_norm", -1.0, "max_norm"),
                              ("max_norm", float("nan"), "max_norm"), ("eps", -1.0, "eps"), ("norm", None, "norm"), ("norm", FAKE + 2, "norm"),
                              ("workspace", None, "workspace"), ("workspace_bytes", 24, "workspace"), ("workspace", FAKE + 8, "aligned")):
        a, keep = clip_block()
        setattr(a, field, value)
        refused(a, nat.SS_ERR_INVALID, msg)
    for i, value, code, msg in ((0, FAKE + 1, nat.SS_ERR_INVALID, "misaligned"), (0, None, nat.SS_ERR_INVALID, "NULL"),
                                (2, -3, nat.SS_ERR_INVALID, "negative size"), (2, 1 << 41, nat.SS_ERR_UNSUPPORTED, "2^40"),
                                (3, 4, nat.SS_ERR_INVALID, "dtype")):
        a, keep = clip_block()
        keep[i][1] = value
        refused(a, code, msg)
        assert lib.ss_clip_grads_workspace_bytes(ctypes.byref(a)) == -1
    a, keep = clip_block()
    assert lib.ss_clip_grads_workspace_bytes(ctypes.byref(a)) >= 8
    assert lib.ss_clip_grads(None, None) == nat.SS_ERR_INVALID


def test_cpu_tensors_refused():
    t, w = torch.zeros(3, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="ROCm"):
        block_norm_fn(t, t, w, w)
    with pytest.raises(ValueError, match="ROCm"):
        gated_rms_norm_fn(t, t, w, 2)
    with pytest.raises(ValueError, match="ROCm"):
        clip_grads([t], 1.0)
    with pytest.raises(ValueError, match="out holds"):
        clip_grads([t], 1.0, out=[])


def test_closed_forms_against_differences():
    gen = torch.Generator().manual_seed(0)

    def rand(*s):
        return torch.randn(s, generator=gen, dtype=torch.float64)

    x = {"x": rand(3, 8), "res": rand(3, 8), "post": rand(8), "pre": rand(8), "gate": rand(3, 8), "scale": rand(8)}
    up = rand(3, 8), rand(3, 8)

    def value(y):
        r, _ = border(**y, eps=1e-3)
        return float((r["out"] * up[0] + r["s"] * up[1]).sum())

    got, _ = border(**x, eps=1e-3, dout=up[0], ds=up[1])
    h = 1e-5
    for n in x:
        d = rand(*x[n].shape)
        slope = (value({**x, n: x[n] + h * d}) - value({**x, n: x[n] - h * d})) / (2 * h)
        assert abs(slope - float((got["d" + n] * d).sum())) < 1e-7 * (1 + abs(slope)), n
    y = {"x": x["x"], "gate": x["gate"], "w": x["post"]}

    def value_h(y):
        return float((heads(**y, groups=2, eps=1e-3)[0]["out"] * up[0]).sum())

    got, _ = heads(**y, groups=2, eps=1e-3, dout=up[0])
    for n, g in (("x", "dx"), ("gate", "dgate"), ("w", "dweight")):
        d = rand(*y[n].shape)
        slope = (value_h({**y, n: y[n] + h * d}) - value_h({**y, n: y[n] - h * d})) / (2 * h)
        assert abs(slope - float((got[g] * d).sum())) < 1e-7 * (1 + abs(slope)), n


def test_struct_layout_matches_c_compiler(tmp_path):
    structs = ((nat.BlockNormArgs, "ss_block_norm_args"), (nat.BlockNormBwdArgs, "ss_block_norm_bwd_args"),
               (nat.GatedNormArgs, "ss_gated_norm_args"), (nat.GatedNormBwdArgs, "ss_gated_norm_bwd_args"),
               (nat.ClipGradsArgs, "ss_clip_grads_args"))
    body = "".join(f'printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for T, n in structs for f, _ in T._fields_)
    body += "".join(f'printf("{n} size %zu\\n", sizeof({n}));' for _, n in structs)
    src = tmp_path / "probe.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "mamba_ss.h"\nint main(void) {{ {body} return 0; }}\n')
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", inc, str(src), "-o", str(tmp_path / "probe")], check=True)
    lines = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.splitlines()
    got = {tuple(l.split()[:2]): int(l.split()[2]) for l in lines}
    for T, n in structs:
        assert got[(n, "size")] == ctypes.sizeof(T), n
        for f, _ in T._fields_:
            assert got[(n, f)] == getattr(T, f).offset, (n, f)
