from omnistack_rs.attention.prompt import prompt_attention
from omnistack_rs.attention.reference import ReferenceAttention, reference_attn, repeat_kv

__all__ = ["ReferenceAttention", "prompt_attention", "reference_attn", "repeat_kv"]
