"""Refusals of the gated delta rule: argument blocks through the C ABI and tensors
through Python, no device work; and the float64 recurrence's own gradients against
differences."""
import ctypes

import pytest
import torch

from mamba_amd import _native as nat
from mamba_amd.ops.delta_rule import delta_rule_fn, delta_rule_update
from tests._delta_rule_ref import recurrence

FAKE = 1 << 20   # aligned, never dereferenced


def block(cls=nat.DeltaRuleArgs):
    a = nat.DeltaRuleArgs()
    a.batch, a.seqlen, a.heads, a.groups, a.d_key, a.d_value = 2, 100, 4, 2, 64, 48
    a.dtype, a.scale = nat.SS_BF16, 0.125
    for i, n in enumerate(("q", "k", "v", "g", "beta", "out")):
        setattr(a, n, FAKE + 4096 * i)
    if cls is nat.DeltaRuleArgs:
        return a
    b = nat.DeltaRuleBwdArgs()
    b.f = a
    b.f.saved, b.f.saved_bytes = FAKE, 1 << 40
    for i, n in enumerate(("dout", "dq", "dk", "dv", "dg", "dbeta")):
        setattr(b, n, FAKE + 65536 + 4096 * i)
    return b


BREAKS = [
    ("batch", -1, "INVALID", "negative size"), ("dtype", 9, "INVALID", "dtype"), ("d_key", 0, "UNSUPPORTED", "d_key"),
    ("d_key", 257, "UNSUPPORTED", "d_key"), ("d_value", 300, "UNSUPPORTED", "d_value"), ("groups", 3, "INVALID", "multiple of groups"),
    ("groups", 0, "INVALID", "multiple of groups"), ("q", None, "INVALID", "NULL"), ("beta", None, "INVALID", "NULL"),
    ("v", FAKE + 1, "INVALID", "misaligned"), ("beta", FAKE + 2, "INVALID", "misaligned"), ("beta_len_stride", -1, "INVALID", "stride"),
    ("seqlen", 1 << 25, "UNSUPPORTED", "seqlen"), ("batch", 1 << 40, "UNSUPPORTED", "too large"),
    ("lengths", FAKE + 2, "INVALID", "lengths"),
]


@pytest.mark.parametrize("field,value,code,msg", BREAKS, ids=[f"{b[0]}={b[1]}" for b in BREAKS])
def test_blocks_refused(field, value, code, msg):
    lib = nat.load()
    a, b = block(), block(nat.DeltaRuleBwdArgs)
    setattr(a, field, value)
    setattr(b.f, field, value)
    want = getattr(nat, f"SS_ERR_{code}")
    for fn, arg in ((lib.ss_delta_rule_fwd, a), (lib.ss_delta_rule_bwd, b)):
        assert fn(ctypes.byref(arg), None) == want and msg in lib.ss_last_error().decode()
    assert lib.ss_delta_rule_saved_bytes(ctypes.byref(a)) == -1
    assert lib.ss_delta_rule_fwd_workspace_bytes(ctypes.byref(a)) == -1
    assert lib.ss_delta_rule_bwd_workspace_bytes(ctypes.byref(b)) == -1


def test_launches_too_large():
    lib = nat.load()
    a = block()
    a.batch, a.heads, a.seqlen = 1 << 10, 1 << 10, 1 << 10
    assert lib.ss_delta_rule_fwd(ctypes.byref(a), None) == nat.SS_ERR_UNSUPPORTED and "too large" in lib.ss_last_error().decode()


def test_spaces_refused():
    lib = nat.load()
    a = block()
    need = lib.ss_delta_rule_fwd_workspace_bytes(ctypes.byref(a))
    assert need > 0
    for ws, n in ((None, 0), (FAKE, need - 1), (FAKE + 8, need)):
        a.workspace, a.workspace_bytes = ws, n
        assert lib.ss_delta_rule_fwd(ctypes.byref(a), None) == nat.SS_ERR_INVALID and "workspace" in lib.ss_last_error().decode()
    a = block()
    n = lib.ss_delta_rule_saved_bytes(ctypes.byref(a))
    a.saved, a.saved_bytes = FAKE, n - 1
    assert lib.ss_delta_rule_fwd(ctypes.byref(a), None) == nat.SS_ERR_INVALID and "saved" in lib.ss_last_error().decode()
    for saved, size in ((None, 0), (FAKE, n - 1), (FAKE + 8, n)):
        b = block(nat.DeltaRuleBwdArgs)
        b.f.saved, b.f.saved_bytes = saved, size
        assert lib.ss_delta_rule_bwd(ctypes.byref(b), None) == nat.SS_ERR_INVALID and "saved" in lib.ss_last_error().decode()
    b = block(nat.DeltaRuleBwdArgs)
    need = lib.ss_delta_rule_bwd_workspace_bytes(ctypes.byref(b))
    for ws, size in ((None, 0), (FAKE, need - 1)):
        b.f.workspace, b.f.workspace_bytes = ws, size
        assert lib.ss_delta_rule_bwd(ctypes.byref(b), None) == nat.SS_ERR_INVALID and "workspace" in lib.ss_last_error().decode()
    for field in ("dout", "dq", "dg", "dbeta"):
        b = block(nat.DeltaRuleBwdArgs)
        setattr(b, field, None)
        assert lib.ss_delta_rule_bwd(ctypes.byref(b), None) == nat.SS_ERR_INVALID and "NULL" in lib.ss_last_error().decode()
    for fn in (lib.ss_delta_rule_fwd, lib.ss_delta_rule_bwd, lib.ss_delta_rule_update):
        assert fn(None, None) == nat.SS_ERR_INVALID


def test_update_block_refused():
    lib = nat.load()
    for field, value, msg in (("d_key", 257, "d_key"), ("groups", 3, "multiple"), ("dtype", 5, "dtype"), ("state", None, "NULL"),
                              ("beta", None, "NULL"), ("state", FAKE + 2, "misaligned"), ("beta_head_stride", -2, "stride"),
                              ("heads", -1, "negative size"), ("state_head_stride", 64, "overlap"), ("out_batch_stride", 64, "overlap")):
        a = nat.DeltaRuleUpdateArgs()
        a.batch, a.heads, a.groups, a.d_key, a.d_value, a.dtype = 2, 4, 2, 64, 64, nat.SS_F32
        a.state_batch_stride, a.state_head_stride, a.out_batch_stride, a.out_head_stride = 4 * 4096, 4096, 256, 64
        for i, n in enumerate(("state", "q", "k", "v", "g", "beta", "out")):
            setattr(a, n, FAKE + 4096 * i)
        setattr(a, field, value)
        assert lib.ss_delta_rule_update(ctypes.byref(a), None) != nat.SS_OK and msg in lib.ss_last_error().decode(), field


def test_cpu_tensors_refused():
    t, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    with pytest.raises(ValueError, match="ROCm"):
        delta_rule_fn(t, t, t, g, g)
    with pytest.raises(ValueError, match="ROCm"):
        delta_rule_update(torch.zeros(1, 2, 8, 8), t[:, 0], t[:, 0], t[:, 0], g[:, 0], g[:, 0])


def test_recurrence_gradients():
    """The float64 recurrence's gradients against central differences (the oracle of the GPU tests)."""
    gen = torch.Generator().manual_seed(0)

    def rand(*s):
        return torch.randn(s, generator=gen, dtype=torch.float64)

    x = {"q": rand(2, 6, 1, 3), "k": rand(2, 6, 1, 3) * 0.5, "v": rand(2, 6, 2, 4), "g": -rand(2, 6, 2).abs(),
         "beta": torch.sigmoid(rand(2, 6, 2)), "initial": rand(2, 2, 3, 4)}
    do, dl, n = rand(2, 6, 2, 4), rand(2, 2, 3, 4), torch.tensor([6, 4])

    def value(y):
        r = recurrence(y["q"], y["k"], y["v"], y["g"], y["beta"], 0.7, y["initial"], n)
        return float((r["out"] * do).sum() + (r["last"] * dl).sum())

    r = recurrence(x["q"], x["k"], x["v"], x["g"], x["beta"], 0.7, x["initial"], n, do, dl)
    for name in x:
        d = rand(*x[name].shape)
        if name != "initial":
            d[1, 4:] = 0.0
        h = 1e-5
        slope = (value({**x, name: x[name] + h * d}) - value({**x, name: x[name] - h * d})) / (2 * h)
        assert abs(slope - float((r["d" + name] * d).sum())) < 1e-7 * (1 + abs(slope)), name


def test_struct_layout_matches_c_compiler(tmp_path):
    import os
    import subprocess
    structs = ((nat.DeltaRuleArgs, "ss_delta_rule_args"), (nat.DeltaRuleBwdArgs, "ss_delta_rule_bwd_args"),
               (nat.DeltaRuleUpdateArgs, "ss_delta_rule_update_args"))
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
