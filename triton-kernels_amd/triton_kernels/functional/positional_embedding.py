"""Plain-PyTorch RoPE application (functional/positional_embedding.py:5-10 of the reference): every
adjacent pair (x[2i], x[2i+1]) is multiplied by the 2x2 matrix freqs_cis[..., i, :, :]."""
import torch
from torch import Tensor


def _rotate(x: Tensor, freqs_cis: Tensor) -> Tensor:
    pairs = x.float().unflatten(-1, (-1, 1, 2))          # [..., D/2, 1, 2]
    out = freqs_cis[..., 0] * pairs[..., 0] + freqs_cis[..., 1] * pairs[..., 1]
    return out.flatten(-2).type_as(x)


def apply_rope_torch(xq: Tensor, xk: Tensor, freqs_cis: Tensor) -> tuple[Tensor, Tensor]:
    return _rotate(xq, freqs_cis), _rotate(xk, freqs_cis)


apply_rope_torch_compile = apply_rope_torch


def apply_rope_nd_torch(xq: Tensor, xk: Tensor, ids: Tensor, axes_dim, theta: float = 10000.0) -> tuple[Tensor, Tensor]:
    """Rotation by positions of several axes: angles in float64, the rotation in float32, rounded once."""
    dims = torch.tensor(list(axes_dim), device=ids.device)
    axis = torch.repeat_interleave(torch.arange(len(dims), device=ids.device), dims // 2)
    place = torch.arange(len(axis), device=ids.device) - (torch.cumsum(dims // 2, 0) - dims // 2)[axis]
    angle = ids.double()[..., axis] * theta ** (-2.0 * place.double() / dims[axis].double())
    c, s = torch.cos(angle).float().unsqueeze(-3), torch.sin(angle).float().unsqueeze(-3)
    return apply_rope_torch(xq, xk, torch.stack((c, -s, s, c), dim=-1).unflatten(-1, (2, 2)))
