from .causal_lm import Block, CausalLM, CausalLMConfig, GraphedStep
from .linear_attn_lm import LinearAttnLM, LinearAttnLMConfig

__all__ = ["Block", "CausalLM", "CausalLMConfig", "GraphedStep", "LinearAttnLM", "LinearAttnLMConfig"]
