"""The packages export their operators, modules and models, and leave their submodules reachable by name."""
import importlib

import pytest


@pytest.mark.parametrize("package,names", [
    ("ops", ["selective_scan_fn", "SelectiveScanFn", "linear_attn_fn", "linear_attn_update", "block_norm_fn", "gated_rms_norm_fn"]),
    ("modules", ["MambaSimple", "RMSNorm", "LinearAttn"]),
    ("models", ["CausalLM", "CausalLMConfig", "GraphedStep", "Block", "LinearAttnLM", "LinearAttnLMConfig"])])
def test_exports(package, names):
    m = importlib.import_module(f"mamba_amd.{package}")
    assert set(names) == set(m.__all__)
    for n in names:
        assert callable(getattr(m, n))


def test_submodules_keep_their_names():
    from mamba_amd.ops import block_norm, clip_grads, linear_attn
    for m, n in ((block_norm, "block_norm_fn"), (clip_grads, "clip_grads"), (linear_attn, "linear_attn_fn")):
        assert callable(getattr(m, n)) and m.__name__.startswith("mamba_amd.ops.")
