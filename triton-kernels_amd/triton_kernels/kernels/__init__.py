"""Operator entry points: thin Python launchers over the C ABI of libfluxhip.so. They hand addresses and streams to the library, which
torch.compile cannot follow: in code that it traces, each runs by itself between two compiled parts (a graph break; fullgraph=True refuses it)."""
from triton_kernels.kernels.normalization import layer_norm, layer_norm_modulation, rms_norm
from triton_kernels.kernels.positional_embedding import apply_rope, apply_rope_nd, qkv_prep, rope_table
from triton_kernels.kernels.linear import linear, linear_into, linear_lora, linear_w4, qk_fusable
from triton_kernels.kernels.quantization import W4, pack_w4, quantize_w4
from triton_kernels.kernels.attention import attention_into, block_sparse_attention, scaled_dot_product_attention, select_blocks

__all__ = [
    "apply_rope", "layer_norm", "layer_norm_modulation", "linear", "rms_norm", "scaled_dot_product_attention",
    "apply_rope_nd", "qkv_prep", "rope_table", "linear_into", "linear_lora", "linear_w4", "attention_into",
    "W4", "pack_w4", "quantize_w4", "block_sparse_attention", "select_blocks",
]
