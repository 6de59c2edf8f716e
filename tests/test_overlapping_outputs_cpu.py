"""In-place and output tensors whose elements overlap are refused: several
workgroups would write one element.  The rule (csrc/overlap.hpp) built for the host and
tried against all pairs of blocks, and argument blocks through the C ABI, no
device work."""
import ctypes
import os
import shutil
import subprocess

import pytest

from mamba_amd import _native as nat

FAKE = 1 << 20   # aligned, never dereferenced
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba_amd", "csrc")
PROGRAM = """
#include <cstdio>
#include <cstdlib>
#include "overlap.hpp"
int main() {
    int bad = 0;
    for (int64_t size : {1, 2, 5})
        for (int64_t n1 = 1; n1 <= 4; ++n1)
            for (int64_t n2 = 1; n2 <= 5; ++n2)
                for (int64_t s1 = 0; s1 <= 30; ++s1)
                    for (int64_t s2 = 0; s2 <= 30; ++s2) {
                        bool want = false;
                        for (int64_t a = 0; a < n1 * n2; ++a)
                            for (int64_t b = 0; b < a; ++b)
                                want |= std::llabs(a / n2 * s1 + a % n2 * s2 - b / n2 * s1 - b % n2 * s2) < size;
                        if (ss::blocks_overlap(n1, s1, n2, s2, size) != want)
                            ++bad, std::printf("%ld x %ld, strides %ld %ld, size %ld\\n", n1, n2, s1, s2, size);
                    }
    const int64_t far = INT64_MAX;                     // offsets past 64 bits
    bad += ss::blocks_overlap(2, far, 1 << 10, far - 100, 4) || !ss::blocks_overlap(2, far, 1 << 10, far - 3, 4);
    bad += ss::blocks_overlap(1 << 20, far / 2, 1, 0, 65536) || ss::blocks_overlap(0, 0, 7, 0, 9) || ss::blocks_overlap(7, 0, 7, 0, 0);
    bad += !ss::blocks_overlap(1 << 10, far, 1 << 10, far, 4);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_the_rule(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout[-2000:]


# (batch, heads, strides): one state for all rows or all heads, blocks too close, dims that interleave
@pytest.mark.parametrize("batch,heads,strides", [(4, 5, (0, 0)), (4, 5, (0, 1)), (4, 5, (5, 0)), (4, 1, (0, 1)), (1, 5, (0, 0)), (4, 5, (1, 1)),
                                                 (4, 5, (3, 2))], ids=str)
@pytest.mark.parametrize("which", ["state", "out"])
def test_update_refused(which, batch, heads, strides):
    lib = nat.load()
    a = nat.LinearAttnUpdateArgs()
    a.batch, a.heads, a.groups, a.d_key, a.d_value, a.dtype = batch, heads, 1, 8, 6, nat.SS_F32
    for n, size in (("state", 48), ("out", 6)):
        b, h = strides if n == which else (heads, 1)
        setattr(a, n + "_batch_stride", b * size)
        setattr(a, n + "_head_stride", h * size)
    for i, n in enumerate(("state", "q", "k", "v", "g", "out")):
        setattr(a, n, FAKE + 65536 * i)
    assert lib.ss_linear_attn_update(ctypes.byref(a), None) == nat.SS_ERR_INVALID
    assert f"{which}'s elements overlap" in lib.ss_last_error().decode()


SPANS = """
#include <cstdio>
#include <cstdlib>
#include "overlap.hpp"
int main() {
    int bad = 0;
    std::srand(1);
    for (int turn = 0; turn < 200000; ++turn) {
        std::vector<ss::Span> ins, outs;
        const int n = 1 + std::rand() % 4;
        for (int64_t i = 0; i < n; ++i) {
            const uintptr_t size = 1 + std::rand() % 6, in = std::rand() % 40;
            const uintptr_t out = std::rand() % 3 ? in : std::rand() % 40;
            if (in != out) ins.push_back({in, in + size, i});
            outs.push_back({out, out + size, i});
        }
        bool want = false;
        const auto meet = [](const ss::Span& a, const ss::Span& b) { return a.from < b.to && b.from < a.to; };
        for (size_t i = 0; i < outs.size(); ++i) {
            for (size_t j = 0; j < i; ++j) want |= meet(outs[i], outs[j]);
            for (const ss::Span& in : ins) want |= meet(outs[i], in);
        }
        const int64_t at = ss::outputs_clash(ins, outs);
        if ((at >= 0) != want || at >= n) ++bad, std::printf("turn %d\\n", turn);
    }
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_the_rule_of_spans(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(SPANS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout[-2000:]


# (grads, outs) as offsets in bytes of two tensors of 100 bf16 elements: one tensor twice, two that overlap, an output
# over another's gradient, one that slides over its own
@pytest.mark.parametrize("grads,outs", [((0, 0), (0, 0)), ((0, 198), (0, 198)), ((0, 0), (4096, 4096)), ((0, 4096), (4096, 8192)),
                                        ((0, 4096), (2, 8192)), ((8192, 4096), (0, 4294))], ids=str)
def test_clip_refused(grads, outs):
    lib = nat.load()
    a = nat.ClipGradsArgs()
    a.count, a.max_norm, a.eps, a.norm, a.workspace, a.workspace_bytes = 2, 1.0, 1e-6, FAKE, FAKE, 1 << 20
    keep = ((ctypes.c_void_p * 2)(*(2 * FAKE + x for x in grads)), (ctypes.c_void_p * 2)(*(2 * FAKE + x for x in outs)),
            (ctypes.c_int64 * 2)(100, 100), (ctypes.c_int32 * 2)(nat.SS_BF16, nat.SS_BF16))
    a.grads, a.outs, a.numels, a.dtypes = (ctypes.cast(k, ctypes.c_void_p) for k in keep)
    assert lib.ss_clip_grads(ctypes.byref(a), None) == nat.SS_ERR_INVALID
    assert "lies over another tensor" in lib.ss_last_error().decode()
