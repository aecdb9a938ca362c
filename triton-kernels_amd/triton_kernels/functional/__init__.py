from triton_kernels.functional.attention import block_sparse_attention_torch, select_blocks_torch
from triton_kernels.functional.linear import linear_lora_torch, linear_w4_torch
from triton_kernels.functional.normalization import (
    layer_norm_modulation_torch,
    layer_norm_modulation_torch_compile,
    layer_norm_torch,
    modulate,
    rms_norm_torch,
    rms_norm_torch_compile,
)
from triton_kernels.functional.positional_embedding import apply_rope_nd_torch, apply_rope_torch, apply_rope_torch_compile

__all__ = [
    "apply_rope_nd_torch", "apply_rope_torch", "apply_rope_torch_compile", "layer_norm_modulation_torch",
    "layer_norm_modulation_torch_compile", "layer_norm_torch", "linear_lora_torch", "linear_w4_torch", "block_sparse_attention_torch", "select_blocks_torch", "modulate", "rms_norm_torch", "rms_norm_torch_compile",
]
