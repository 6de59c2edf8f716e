from .linear_attn import LinearAttn
from .mamba_simple import MambaSimple
from .rms_norm import RMSNorm

__all__ = ["LinearAttn", "MambaSimple", "RMSNorm"]
