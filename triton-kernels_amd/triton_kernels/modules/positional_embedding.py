"""EmbedND (flux/layers.py:38-52 of the reference) on the HIP rope_table: the rotation table of the blocks in one kernel."""
from torch import Tensor, nn

from triton_kernels.kernels.positional_embedding import rope_table


class EmbedND(nn.Module):
    """ids [B, L, n_axes] -> fp32 [B, 1, L, sum(axes_dim) / 2, 2, 2]."""

    def __init__(self, dim: int, theta: int, axes_dim: list[int]):
        super().__init__()
        self.dim, self.theta, self.axes_dim = dim, theta, list(axes_dim)

    def forward(self, ids: Tensor) -> Tensor:
        return rope_table(ids, self.axes_dim, self.theta)
