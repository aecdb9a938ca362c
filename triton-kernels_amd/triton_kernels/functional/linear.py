"""Plain-PyTorch statements of the projections with adapters and with weights in 4 bits: float32 throughout, rounded once."""
import torch
import torch.nn.functional as F
from torch import Tensor


def linear_lora_torch(x: Tensor, w: Tensor, b: Tensor | None, lora_a: Tensor, lora_b: Tensor, adapter: Tensor, scaling: Tensor | None = None, activation: str = "") -> Tensor:
    y = x.float() @ w.float().T
    if b is not None:
        y = y + b.float()
    rows = y.view(*adapter.shape, -1, w.shape[0])
    xs = x.float().reshape(*adapter.shape, -1, x.shape[-1])
    for i in range(lora_a.shape[0]):
        at = adapter == i
        s = 1.0 if scaling is None else scaling[i].float()
        rows[at] = rows[at] + s * ((xs[at] @ lora_a[i].float().T) @ lora_b[i].float().T)
    return (F.gelu(y, approximate="tanh") if activation == "GELU" else y).to(x.dtype)


def linear_w4_torch(x: Tensor, q: Tensor, scale: Tensor, zero: Tensor | None = None, b: Tensor | None = None, activation: str = "", in_activation: str = "") -> Tensor:
    """The weight as pack_w4 takes it: w[n, k] = (q[n, k] - zero[n, k / group]) * scale[n, k / group]."""
    offset = 8.0 if zero is None else zero.float()[..., None]
    w = ((q.float().unflatten(1, (scale.shape[1], -1)) - offset) * scale.float()[..., None]).flatten(1)
    xf = F.silu(x.float()) if in_activation == "SiLU" else x.float()
    y = xf @ w.T
    if b is not None:
        y = y + b.float()
    return (F.gelu(y, approximate="tanh") if activation == "GELU" else y).to(x.dtype)
