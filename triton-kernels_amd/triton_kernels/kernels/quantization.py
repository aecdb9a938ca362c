"""Weights held in 4 bits, a scale and (or not) a zero point for each group of columns, as linear_w4 takes them: pack_w4 and
quantize_w4 lay them out. The reference has nothing of this kind."""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from triton_kernels import _native as nv

GROUPS = (32, 64, 128)
_TILE, _CHUNK = 16, 128


@dataclass(frozen=True)
class W4:
    """A weight [N, K] in 4 bits, w = (q - zero) * scale, as the kernels read it (include/flux_hip_serve.h has the layout).

    packed : uint8 [N / 16, K / 128, 1024], scale : bf16 [N / 16, K / 128, 16, 128 / group], zero : the same in uint8, or None for 8; N and K
             rounded up to whole tiles
    shape  : (N, K), group : columns that share a scale
    """

    packed: Tensor
    scale: Tensor
    zero: Tensor | None
    shape: tuple[int, int]
    group: int

    def __post_init__(self):
        n, k = self.shape
        assert self.group in GROUPS, f"groups of {GROUPS} columns, not {self.group}"
        assert n >= 0 and k >= 0 and k % self.group == 0, f"{k} columns are not whole groups of {self.group}"
        tiles = (-(-n // _TILE), -(-k // _CHUNK))
        assert self.packed.dtype == torch.uint8 and self.packed.shape == (*tiles, _TILE * _CHUNK // 2) and self.packed.is_contiguous(), "packed is laid out by pack_w4"
        for t, dtype in ((self.scale, torch.bfloat16), (self.zero, torch.uint8)):
            assert t is None or (t.dtype == dtype and t.shape == (*tiles, _TILE, _CHUNK // self.group) and t.is_contiguous()), "scale and zero are laid out by pack_w4"
        assert self.scale is not None, "scale is laid out by pack_w4"

    @classmethod
    def zeros(cls, n: int, k: int, group: int = 64, zero_points: bool = False, device=None) -> "W4":
        """A weight of zeros: scales of 0."""
        assert group in GROUPS and k % group == 0, f"{k} columns are not whole groups of {GROUPS}"
        tiles = (-(-n // _TILE), -(-k // _CHUNK))
        numbers = (*tiles, _TILE, _CHUNK // group)
        return cls(torch.zeros(*tiles, _TILE * _CHUNK // 2, dtype=torch.uint8, device=device), torch.zeros(numbers, dtype=torch.bfloat16, device=device),
                   torch.zeros(numbers, dtype=torch.uint8, device=device) if zero_points else None, (n, k), group)

    def to(self, device) -> "W4":
        return W4(self.packed.to(device), self.scale.to(device), None if self.zero is None else self.zero.to(device), self.shape, self.group)

    def unpack(self) -> tuple[Tensor, Tensor, Tensor | None]:
        """q (uint8 [N, K]), scale and zero ([N, K / group]) as pack_w4 takes them."""
        (n, k), (rows, chunks) = self.shape, self.packed.shape[:2]
        words = self.packed.view(rows, chunks, 4, _TILE, 4, 4)   # [.., g, row, j, byte]: elements 2i and 2i + 1 of a word at bits 4i and 16 + 4i
        nibbles = torch.stack((words & 15, words >> 4), -1).flatten(-2)   # by bit: elements 0, 2, 4, 6, 1, 3, 5, 7
        q = nibbles.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-2)   # [.., g, row, j, e]
        q = q.permute(0, 3, 1, 4, 2, 5).reshape(rows * _TILE, chunks * _CHUNK)[:n, :k]

        def by_group(t):
            return None if t is None else t.transpose(1, 2).reshape(rows * _TILE, chunks * (_CHUNK // self.group))[:n, :k // self.group].contiguous()

        return q.contiguous(), by_group(self.scale), by_group(self.zero)

    def dequantize(self) -> Tensor:
        """The weight as bf16 [N, K], each value rounded once."""
        dev = nv.require_gpu(self.packed, self.scale, self.zero)
        out = torch.empty(self.shape, dtype=torch.bfloat16, device=dev)
        if out.numel():
            with nv.on_device(dev):
                nv.check(nv.lib().flux_w4_unpack(nv.byref(self._args()), out.data_ptr(), nv.stream_ptr(dev)), "flux_w4_unpack")
        return out

    def _args(self) -> "nv.W4":
        return nv.W4(self.packed.data_ptr(), self.scale.data_ptr(), nv.ptr(self.zero), *self.shape, self.group)


def pack_w4(q: Tensor, scale: Tensor, zero: Tensor | None = None) -> W4:
    """Lays a weight out for linear_w4, once; on any device.

    q     : whole numbers 0 .. 15, [N, K]
    scale : bf16 [N, K / group], group 32, 64 or 128: w[n, k] = (q[n, k] - zero[n, k / group]) * scale[n, k / group]
    zero  : whole numbers 0 .. 15, [N, K / group], or None for 8
    """
    assert q.dim() == 2 and scale.dim() == 2 and scale.shape[0] == q.shape[0] and scale.shape[1] > 0, f"q is [N, K] and scale [N, K / group], not {tuple(q.shape)} and {tuple(scale.shape)}"
    n, k = q.shape
    group = k // scale.shape[1]
    assert group in GROUPS and group * scale.shape[1] == k, f"{k} columns and {scale.shape[1]} scales are no groups of {GROUPS}"
    if scale.dtype != torch.bfloat16:
        raise TypeError(f"unsupported dtype {scale.dtype} of scales: the kernels take bfloat16")
    for t in (q, zero):
        if t is None:
            continue
        if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
            raise TypeError(f"unsupported dtype {t.dtype} of 4-bit numbers")
        if t.dtype in (torch.uint16, torch.uint32, torch.uint64):   # (these have no smallest and largest; 2^63 and more are below 0 then)
            t = t.to(torch.int64)
        if t.numel() and not 0 <= int(t.min()) <= int(t.max()) <= 15:
            raise ValueError("4-bit numbers are 0 .. 15")
    assert zero is None or zero.shape == scale.shape, f"zero is {tuple(scale.shape)} as scale, not {tuple(zero.shape)}"
    rows, chunks, per = -(-n // _TILE), -(-k // _CHUNK), _CHUNK // group

    def padded(t, width, dtype):
        full = torch.zeros(rows * _TILE, width, dtype=dtype, device=t.device)
        full[:n, :t.shape[1]] = t
        return full.view(rows, _TILE, chunks, width // chunks)

    e = padded(q, chunks * _CHUNK, torch.uint8).view(rows, _TILE, chunks, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)   # [row tile, chunk, g, row, j, e]
    nibbles = e.unflatten(-1, (4, 2)).transpose(-1, -2).flatten(-2)   # by bit of the word: 0, 2, 4, 6, 1, 3, 5, 7
    packed = (nibbles[..., ::2] | nibbles[..., 1::2] << 4).reshape(rows, chunks, _TILE * _CHUNK // 2)
    scales = padded(scale, chunks * per, torch.bfloat16).transpose(1, 2).contiguous()
    zeros = None if zero is None else padded(zero, chunks * per, torch.uint8).transpose(1, 2).contiguous()
    return W4(packed, scales, zeros, (n, k), group)


def quantize_w4(w: Tensor, group: int = 64, zero_points: bool = False) -> W4:
    """Weights in 4 bits from w [N, K]: each group's largest value sets its scale, and with zero_points the range from its smallest to its largest value
    (0 among them) does. q is the nearest whole number; a group of zeros has scale 0. Values that are not finite are refused."""
    assert w.dim() == 2 and group in GROUPS and w.shape[1] > 0 and w.shape[1] % group == 0, f"w is [N, K] with whole groups of {GROUPS} columns, not {tuple(w.shape)} in {group}"
    wf = w.detach().float().unflatten(1, (-1, group))
    if not bool(torch.isfinite(wf).all()):
        raise ValueError("quantize_w4: the weight holds values that are not finite")
    if zero_points:
        low, high = wf.amin(-1).clamp(max=0), wf.amax(-1).clamp(min=0)
        scale = (high / 15 - low / 15).to(torch.bfloat16)   # (their difference may be beyond fp32)
    else:
        scale = (wf.abs().amax(-1) / 7.5).to(torch.bfloat16)
    step = torch.where(scale == 0, 1.0, scale.float())
    zero = torch.round(-low / step).clamp(0, 15) if zero_points else torch.full_like(step, 8)
    q = (torch.round(wf / step[..., None]) + zero[..., None]).clamp(0, 15).flatten(1)
    return pack_w4(q.to(torch.uint8), scale, zero.to(torch.uint8) if zero_points else None)
