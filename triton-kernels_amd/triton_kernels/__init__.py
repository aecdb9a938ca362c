"""triton_kernels: the Flux transformer-block operator set, backed by hand-written HIP kernels for
MI355X (gfx950) in libfluxhip.so. The public names are those of the reference package
(triton_kernels/__init__.py:1-10); nothing here uses Triton."""
from triton_kernels.functional import (
    apply_rope_nd_torch,
    apply_rope_torch,
    apply_rope_torch_compile,
    block_sparse_attention_torch,
    layer_norm_modulation_torch,
    layer_norm_modulation_torch_compile,
    layer_norm_torch,
    linear_lora_torch,
    linear_w4_torch,
    rms_norm_torch,
    rms_norm_torch_compile,
    select_blocks_torch,
)
from triton_kernels.kernels import (
    W4,
    apply_rope,
    apply_rope_nd,
    attention_into,
    block_sparse_attention,
    layer_norm,
    layer_norm_modulation,
    linear,
    linear_into,
    linear_lora,
    linear_w4,
    pack_w4,
    qkv_prep,
    quantize_w4,
    rms_norm,
    rope_table,
    scaled_dot_product_attention,
    select_blocks,
)
from triton_kernels.modules import DoubleStreamBlock, EmbedND, LayerNorm, LinearW4, QKNorm, RMSNorm, SingleStreamBlock

__all__ = [
    "apply_rope_nd_torch", "apply_rope_torch", "apply_rope_torch_compile", "layer_norm_modulation_torch",
    "layer_norm_modulation_torch_compile", "layer_norm_torch", "linear_lora_torch", "linear_w4_torch", "block_sparse_attention_torch", "select_blocks_torch", "rms_norm_torch", "rms_norm_torch_compile",
    "apply_rope", "apply_rope_nd", "layer_norm", "layer_norm_modulation", "linear", "rms_norm", "scaled_dot_product_attention",
    "attention_into", "linear_into", "linear_lora", "linear_w4", "qkv_prep", "rope_table", "W4", "pack_w4", "quantize_w4", "block_sparse_attention", "select_blocks",
    "DoubleStreamBlock", "EmbedND", "LayerNorm", "LinearW4", "QKNorm", "RMSNorm", "SingleStreamBlock",
]
