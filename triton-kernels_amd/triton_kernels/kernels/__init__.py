"""Operator entry points: thin Python launchers over the C ABI of libfluxhip.so. They hand addresses and streams to the library, which
torch.compile cannot follow: in code that it traces, each runs by itself between two compiled parts (a graph break; fullgraph=True refuses it)."""
from triton_kernels.kernels.normalization import layer_norm, layer_norm_modulation, rms_norm
from triton_kernels.kernels.positional_embedding import apply_rope, apply_rope_nd, qkv_prep, rope_table
from triton_kernels.kernels.linear import linear, linear_into, linear_lora, qk_fusable
from triton_kernels.kernels.attention import attention_into, scaled_dot_product_attention

__all__ = [
    "apply_rope", "layer_norm", "layer_norm_modulation", "linear", "rms_norm", "scaled_dot_product_attention",
    "apply_rope_nd", "qkv_prep", "rope_table", "linear_into", "linear_lora", "attention_into",
]
