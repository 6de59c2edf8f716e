from .block_norm import block_norm_fn, gated_rms_norm_fn
from .linear_attn import linear_attn_fn, linear_attn_update
from .selective_scan_interface import SelectiveScanFn, selective_scan_fn

__all__ = ["SelectiveScanFn", "selective_scan_fn", "linear_attn_fn", "linear_attn_update", "block_norm_fn", "gated_rms_norm_fn"]
