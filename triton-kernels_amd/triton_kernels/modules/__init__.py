from triton_kernels.modules.blocks import (
    MLP,
    DoubleStreamBlock,
    Linear,
    LinearGELU,
    LinearW4,
    Modulation,
    ModulationOut,
    SelfAttention,
    SingleStreamBlock,
    attention,
)
from triton_kernels.modules.normalization import LayerNorm, QKNorm, RMSNorm
from triton_kernels.modules.positional_embedding import EmbedND

__all__ = [
    "MLP", "DoubleStreamBlock", "Linear", "LinearGELU", "LinearW4", "Modulation", "ModulationOut", "SelfAttention",
    "SingleStreamBlock", "attention", "EmbedND", "LayerNorm", "QKNorm", "RMSNorm",
]
