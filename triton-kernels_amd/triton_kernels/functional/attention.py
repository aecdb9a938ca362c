"""Plain-PyTorch statements of the selection of blocks (float64: which of two neighbours is chosen must not go with rounding) and of attention over
listed blocks (float32, rounded once)."""
import math

import torch
from torch import Tensor

_QUERIES, _KEYS = 128, 64   # of a block


def _seen(k: Tensor, lengths: Tensor | None) -> Tensor:
    """[B, L]: the keys (or queries) that are there."""
    end = torch.full((k.shape[0],), k.shape[2], device=k.device) if lengths is None else lengths
    return torch.arange(k.shape[2], device=k.device) < end[:, None]


def _block_means(x: Tensor, size: int, seen: Tensor) -> tuple[Tensor, Tensor]:
    """[B, H, blocks, D] and the count of tokens of each block, [B, blocks]."""
    short = -x.shape[2] % size
    rows = torch.where(seen[:, None, :, None], x.double(), 0.0)
    rows = torch.nn.functional.pad(rows, (0, 0, 0, short)).unflatten(2, (-1, size))
    count = torch.nn.functional.pad(seen, (0, short)).unflatten(1, (-1, size)).sum(-1)
    return rows.sum(3) / count.clamp(min=1)[:, None, :, None], count


def select_blocks_torch(q: Tensor, k: Tensor, keep: int, always: int = 0, lengths: Tensor | None = None, q_lengths: Tensor | None = None) -> Tensor:
    mq, queries = _block_means(q, _QUERIES, _seen(q, q_lengths))
    mk, count = _block_means(k, _KEYS, _seen(k, lengths))
    score = mq @ mk.repeat_interleave(q.shape[1] // k.shape[1], 1).transpose(2, 3).contiguous()
    score = torch.where(score.isnan(), -math.inf, score)
    score[..., :always] = math.inf
    keep, blocks = min(keep, score.shape[-1]), score.shape[-1]
    there = ((queries > 0)[:, None, :, None] & (count > 0)[:, None, None]).expand_as(score)
    # those that are there in front, in the order of their scores
    order = torch.argsort(score, dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort(there.gather(-1, order).int(), dim=-1, descending=True, stable=True))[..., :keep]
    chosen = torch.where(there.gather(-1, order), order, blocks).sort(-1).values
    return torch.where(chosen == blocks, -1, chosen).to(torch.int32)


def block_sparse_attention_torch(q: Tensor, k: Tensor, v: Tensor, blocks: Tensor, sm_scale: float | None = None, lengths: Tensor | None = None) -> Tensor:
    per, count = q.shape[1] // k.shape[1], -(-k.shape[2] // _KEYS)
    scale = q.shape[3] ** -0.5 if sm_scale is None else sm_scale
    named = torch.where((blocks >= 0) & (blocks < count), blocks.long(), count)
    times = torch.zeros(*blocks.shape[:3], count + 1, device=q.device).scatter_add_(-1, named, torch.ones_like(named, dtype=torch.float32))
    times = times[..., :count].repeat_interleave(_QUERIES, 2)[:, :, :q.shape[2]].repeat_interleave(_KEYS, 3)[..., :k.shape[2]] * _seen(k, lengths)[:, None, None]
    s = q.float() @ k.float().repeat_interleave(per, 1).transpose(2, 3).contiguous() * scale
    s = torch.where(times > 0, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(times > 0, times * torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    vf = torch.where(_seen(k, lengths)[:, None, :, None], v.float(), 0.0).repeat_interleave(per, 1)
    o = (p @ vf) / p.sum(-1, keepdim=True)
    return torch.where((times > 0).any(-1, keepdim=True), o, 0.0).to(q.dtype)
