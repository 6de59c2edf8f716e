"""Refusals of layer norm and the unit norm through the C ABI, no device work; the LayerNorm module on the CPU."""
import ctypes

import pytest
import torch

from mamba_amd import _native as nat
from mamba_amd.modules.layer_norm import LayerNorm
from mamba_amd.ops.layer_norm import layer_norm_fn
from mamba_amd.ops.unit_norm import unit_norm_fn

FAKE = 1 << 20   # aligned, never dereferenced


def fwd():
    a = nat.LayerNormArgs()
    a.rows, a.dim, a.dtype, a.w_dtype, a.eps = 4, 64, nat.SS_BF16, nat.SS_F32, 1e-5
    for i, n in enumerate(("x", "weight", "out")):
        setattr(a, n, FAKE + 4096 * i)
    return a


def bwd():
    g = nat.LayerNormBwdArgs()
    g.rows, g.dim, g.dtype, g.w_dtype = 4, 64, nat.SS_BF16, nat.SS_F32
    for i, n in enumerate(("s", "weight", "stats", "dout", "dx", "dweight", "workspace")):
        setattr(g, n, FAKE + 4096 * i)
    g.workspace_bytes = 1 << 20
    return g


@pytest.mark.parametrize("field,value,msg", [
    ("rows", -1, "negative size"), ("dim", 16385, "above"), ("dtype", 7, "dtype"), ("w_dtype", nat.SS_F16, "weight dtype"),
    ("weight", None, "weight is NULL"), ("weight", FAKE + 2, "weight is misaligned")])
def test_blocks_refused(field, value, msg):
    lib = nat.load()
    for fn, a in ((lib.ss_layer_norm_fwd, fwd()), (lib.ss_layer_norm_bwd, bwd())):
        setattr(a, field, value)
        assert fn(ctypes.byref(a), None) != nat.SS_OK and msg in lib.ss_last_error().decode()


def test_forward_and_backward_blocks_refused():
    lib = nat.load()
    for field, value, msg in (("x", None, "x is NULL"), ("out", None, "out is NULL"), ("x_row_stride", -1, "stride of x"), ("eps", -1.0, "eps"),
                              ("eps", float("nan"), "eps"), ("residual", FAKE + 1, "residual is misaligned"), ("stats", FAKE + 2, "stats is misaligned")):
        a = fwd()
        setattr(a, field, value)
        assert lib.ss_layer_norm_fwd(ctypes.byref(a), None) == nat.SS_ERR_INVALID and msg in lib.ss_last_error().decode()
    for field, value, msg in (("s", None, "s is NULL"), ("stats", None, "stats is NULL"), ("dx", None, "dx is NULL"), ("dweight", None, "dweight"),
                              ("workspace", None, "workspace"), ("workspace_bytes", 100, "workspace"), ("dout_row_stride", -4, "stride of dout")):
        g = bwd()
        setattr(g, field, value)
        assert lib.ss_layer_norm_bwd(ctypes.byref(g), None) == nat.SS_ERR_INVALID and msg in lib.ss_last_error().decode()
    assert lib.ss_layer_norm_bwd_workspace_bytes(-1, 4) == -1 and lib.ss_layer_norm_bwd_workspace_bytes(4, 16385) == -1
    for fn in (lib.ss_layer_norm_fwd, lib.ss_layer_norm_bwd, lib.ss_unit_norm):
        assert fn(None, None) == nat.SS_ERR_INVALID


def test_unit_norm_block_refused():
    lib = nat.load()
    for field, value, msg in (("rows", -1, "negative"), ("heads", -1, "negative"), ("dim", 16385, "above"), ("dtype", 9, "dtype"), ("x", None, "NULL"),
                              ("x", FAKE + 1, "misaligned"), ("x_head_stride", -1, "stride"), ("dout", FAKE + 1, "misaligned"), ("out", None, "NULL"),
                              ("eps", -1.0, "eps"), ("rows", 1 << 32, "too large")):
        a = nat.UnitNormArgs()
        a.rows, a.heads, a.dim, a.dtype, a.eps = 4, 2, 64, nat.SS_F16, 1e-6
        a.x, a.out = FAKE, FAKE + 4096
        setattr(a, field, value)
        assert lib.ss_unit_norm(ctypes.byref(a), None) != nat.SS_OK and msg in lib.ss_last_error().decode(), field


def test_cpu_tensors_refused():
    t = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="ROCm"):
        layer_norm_fn(t, t[0])
    with pytest.raises(ValueError, match="ROCm"):
        unit_norm_fn(t)


@pytest.mark.parametrize("bias", [True, False])
def test_module_on_the_cpu(bias):
    torch.manual_seed(0)
    m = LayerNorm(48, bias=bias)
    with torch.no_grad():
        for p in m.parameters():
            p.uniform_(-1, 1)
    x, r = torch.randn(2, 3, 5, 48).unbind(0)
    out, s = m(x, r, prenorm=True)
    want = torch.nn.functional.layer_norm(x + r, (48,), m.weight, m.bias, m.eps)
    assert torch.equal(s, x + r) and torch.allclose(out, want, rtol=1e-5, atol=1e-5) and torch.equal(m(x, r), out)


def test_struct_layout_matches_c_compiler(tmp_path):
    import os
    import subprocess
    structs = ((nat.LayerNormArgs, "ss_layer_norm_args"), (nat.LayerNormBwdArgs, "ss_layer_norm_bwd_args"),
               (nat.UnitNormArgs, "ss_unit_norm_args"))
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
