from .block_norm import block_norm_fn, gated_rms_norm_fn
from .delta_rule import delta_rule_fn, delta_rule_update
from .layer_norm import layer_norm_fn
from .linear_attn import linear_attn_fn, linear_attn_update
from .selective_scan_interface import SelectiveScanFn, selective_scan_fn
from .unit_norm import unit_norm_fn

__all__ = ["SelectiveScanFn", "selective_scan_fn", "linear_attn_fn", "linear_attn_update", "block_norm_fn", "gated_rms_norm_fn"]
