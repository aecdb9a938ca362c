"""scaled_dot_product_attention: non-causal flash-attention forward (kernels/attention.py:173-221 of
the reference) on the HIP kernel flux_attention_fwd_bf16. select_blocks and block_sparse_attention, which the reference does not
have, are attention over the blocks of keys that a cheap score selects for each block of queries."""
from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd.forward_ad import unpack_dual
from torch.compiler import is_dynamo_compiling

from triton_kernels import _native as nv
from triton_kernels.kernels.linear import hooked, positional, rows_args


def _bhld_view(t: Tensor) -> Tensor:
    if t.stride(-1) != 1 or any(s % 8 for s in t.stride()[:-1]) or t.data_ptr() % 16:
        t = t.contiguous()
    return t


def _may_cut_keys(BH: int, L: int) -> bool:
    """False where flux_attention_workspace_bytes is known to be 0, so that the call is spared the question (0.4 of
    16 us of host time): keys are cut in two or more parts up to 256 workgroups of 128 rows in all, and sixteen
    tiles of 64 keys are too few to pay for the second launch."""
    return L > 1024 and BH * ((L + 127) // 128) <= 128


def takes_rows(BH: int, L: int, D: int, rows: int, K: int) -> bool:
    """Whether products of `rows` rows in all with K values each run beside an attention (attention_into's `beside`) and not in
    front of it (flux_attention_rows_bf16)."""
    return D == 128 and 64 < L and BH * ((L + 127) // 128) <= 256 and not _may_cut_keys(BH, L) and rows <= 4 and rows * K * 2 <= 48 * 1024


def attention_into(q: Tensor, k: Tensor, v: Tensor, out: Tensor, sm_scale: float | None = None,
                   lse: Tensor | None = None, beside: tuple[dict, ...] = ()) -> Tensor:
    """q,k,v,out are [B,H,L,D] views (bf16, last dim contiguous, any other strides).
    beside: one or two linear_into calls of a few rows (the keyword arguments of each) that have nothing to do with the
    attention; the library runs them beside it in one launch where it can."""
    if is_dynamo_compiling():
        return torch.compiler.disable(attention_into)(q, k, v, out, sm_scale, lse, beside)
    if lse is None and not (beside and hooked()):
        o = nv.ops().attention(q, k, v, sm_scale, out, tuple(positional(**call) for call in beside))
        if o is not None:
            return o
    D = q.shape[-1]
    assert D == k.shape[-1] == v.shape[-1]
    assert D in {16, 32, 64, 128, 256}
    assert q.dim() == 4 and q.shape == k.shape == v.shape == out.shape
    if q.dtype != torch.bfloat16 or k.dtype != q.dtype or v.dtype != q.dtype or out.dtype != q.dtype:
        raise TypeError("scaled_dot_product_attention: the HIP kernel takes bfloat16 q, k, v")
    dev = nv.require_gpu(q, k, v, out, lse)
    if sm_scale is None:
        sm_scale = 1 / math.sqrt(D)
    q, k, v = _bhld_view(q), _bhld_view(k), _bhld_view(v)
    B, H, L, _ = q.shape
    a = nv.AttnArgs()
    a.q, a.k, a.v = nv.src4(q), nv.src4(k), nv.src4(v)
    a.o, a.o_sb, a.o_sh, a.o_sl = out.data_ptr(), out.stride(0), out.stride(1), out.stride(2)
    assert out.stride(3) == 1
    a.lse = nv.ptr(lse)
    a.B, a.H, a.L, a.D, a.sm_scale = B, H, L, D, float(sm_scale)
    with nv.on_device(dev):
        need = nv.lib().flux_attention_workspace_bytes(B, H, L, D) if _may_cut_keys(B * H, L) else 0
        if beside:
            rows, _keep = rows_args(beside, dev)
            ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
            rc = nv.lib().flux_attention_rows_bf16(nv.byref(a), nv.byref(rows), nv.ptr(ws), need, nv.stream_ptr(dev))
        elif need:   # keys cut over several workgroups: partial sums in memory of this launch's stream
            ws = torch.empty((need,), dtype=torch.uint8, device=dev)
            rc = nv.lib().flux_attention_fwd_bf16_ws(nv.byref(a), ws.data_ptr(), need, nv.stream_ptr(dev))
        else:
            rc = nv.lib().flux_attention_fwd_bf16(nv.byref(a), nv.stream_ptr(dev))
    nv.check(rc, "flux_attention_fwd_bf16")
    return out


def scaled_dot_product_attention(q: Tensor, k: Tensor, v: Tensor, sm_scale: float = None) -> Tensor:
    if is_dynamo_compiling():
        return torch.compiler.disable(scaled_dot_product_attention)(q, k, v, sm_scale)
    o = nv.ops().attention(q, k, v, sm_scale)
    if o is not None:
        return o
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    return attention_into(q, k, v, o, sm_scale)


QUERY_BLOCK, KEY_BLOCK = 128, 64


def _lengths(lengths: Tensor | None, batch: int, dev: torch.device, most: int) -> Tensor | None:
    if lengths is None:
        return None
    if lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool:
        raise TypeError(f"unsupported dtype {lengths.dtype} of lengths")
    assert lengths.shape == (batch,), f"lengths are [{batch}], not {tuple(lengths.shape)}"
    if lengths.dtype != torch.int32:
        lengths = lengths.long().clamp(0, most).to(torch.int32)   # (a number beyond 32 bits is a long sequence, not what is left of it)
    return lengths.contiguous()


def _sparse_shapes(name: str, q: Tensor, k: Tensor) -> tuple[int, int, int, int, int, int]:
    assert q.dim() == 4 and k.dim() == 4 and q.shape[0] == k.shape[0] and q.shape[3] == k.shape[3], f"{name}: q is [B, Hq, Lq, D] and k [B, Hk, Lk, D], not {tuple(q.shape)} and {tuple(k.shape)}"
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    assert Hk > 0 and Hq > 0 and Hq % Hk == 0, f"{name}: {Hq} heads of q are no multiple of {Hk} heads of k"
    assert D in (64, 128), f"{name}: heads of 64 or 128, not {D}"
    return B, Hq, Hk, Lq, Lk, D


def select_blocks(q: Tensor, k: Tensor, keep: int, *, always: int = 0, lengths: Tensor | None = None, q_lengths: Tensor | None = None) -> Tensor:
    """The blocks of 64 keys that each block of 128 queries attends to: int32 [B, Hq, ceil(Lq / 128), min(keep, ceil(Lk / 64))].

    q, k      : bf16 [B, Hq, Lq, D] and [B, Hk, Lk, D] views, heads of 64 or 128; Hq is a multiple of Hk, query head h reads key head h // (Hq // Hk).
                Up to 16384 blocks of keys. Each call has memory for the means, 8 D bytes a block and head, and beyond 1024 blocks of keys up to
                64 KB for each of them
    keep      : how many blocks; all of them where there are no more
    always    : the first `always` blocks (as many of them as `keep` has room for) are among them in any case: the text in front of an image
    lengths   : whole numbers [B] on the GPU, or None: keys from lengths[b] on are not there
    q_lengths : the same for q: rows from q_lengths[b] on are in no mean, and a block of none but them names nothing (-1 throughout). None: all Lq rows
                are queries. In a padded batch that attends to itself it is `lengths` once more; without it what the padding holds has a share in the
                list of the block that it shares with the last queries, and a NaN there gives that block the lowest numbers

    A block's score is the product of the queries' mean and the mean of its keys, both formed in 64 bits, so that the choice does not go with rounding; the
    lower number goes first among equals, a NaN comes last. The numbers ascend; where a sequence has fewer blocks, -1 stands behind them. Not differentiated.
    """
    if is_dynamo_compiling():
        return torch.compiler.disable(select_blocks)(q, k, keep, always=always, lengths=lengths, q_lengths=q_lengths)
    blocks = nv.ops().select_blocks(q, k, keep, always, lengths, q_lengths)
    if blocks is not None:
        return blocks
    B, Hq, Hk, Lq, Lk, D = _sparse_shapes("select_blocks", q, k)
    if q.dtype != torch.bfloat16 or k.dtype != q.dtype:
        raise TypeError("select_blocks: the HIP kernel takes bfloat16 q, k")
    keep, always = int(keep), int(always)
    assert keep >= 0 and always >= 0, f"select_blocks: keep and always are counts, not {keep} and {always}"
    dev = nv.require_gpu(q, k, lengths, q_lengths)
    lengths, q_lengths = _lengths(lengths, B, dev, Lk), _lengths(q_lengths, B, dev, Lq)
    q, k = _bhld_view(q.detach()), _bhld_view(k.detach())
    keep, always = (min(n, -(-Lk // KEY_BLOCK)) for n in (keep, always))   # (a count may be beyond what the library's arguments hold)
    blocks = torch.empty((B, Hq, -(-Lq // QUERY_BLOCK), keep), dtype=torch.int32, device=dev)
    if blocks.numel() == 0:
        return blocks
    a = nv.SelectBlocksArgs(nv.src4(q), nv.src4(k), nv.ptr(lengths), blocks.data_ptr(), B, Hq, Hk, Lq, Lk, keep, always, D, nv.ptr(q_lengths))
    with nv.on_device(dev):
        need = nv.lib().flux_select_blocks_workspace_bytes(nv.byref(a))
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
        rc = nv.lib().flux_select_blocks(nv.byref(a), nv.ptr(ws), need, nv.stream_ptr(dev))
    nv.check(rc, "flux_select_blocks")
    return blocks


class _block_sparse_attention(torch.autograd.Function):
    """What operands that require gradients have an edge to: an error, not nothing. Forward-mode derivatives and function transforms are refused as well."""

    @staticmethod
    def forward(ctx, *args):
        return _launch_sparse(*args)

    @staticmethod
    def backward(ctx, do):
        raise NotImplementedError("block_sparse_attention is not differentiated")


def _launch_sparse(q: Tensor, k: Tensor, v: Tensor, blocks: Tensor, sm_scale: float | None, lengths: Tensor | None, out: Tensor | None) -> Tensor:
    B, Hq, Hk, Lq, Lk, D = _sparse_shapes("block_sparse_attention", q, k)
    assert v.shape == k.shape, f"block_sparse_attention: k and v are of one shape, not {tuple(k.shape)} and {tuple(v.shape)}"
    if q.dtype != torch.bfloat16 or k.dtype != q.dtype or v.dtype != q.dtype or (out is not None and out.dtype != q.dtype):
        raise TypeError("block_sparse_attention: the HIP kernel takes bfloat16 q, k, v")
    if blocks.is_floating_point() or blocks.is_complex() or blocks.dtype == torch.bool:
        raise TypeError(f"unsupported dtype {blocks.dtype} of block numbers")
    assert blocks.dim() == 4 and blocks.shape[:3] == (B, Hq, -(-Lq // QUERY_BLOCK)), \
        f"block_sparse_attention: blocks are [{B}, {Hq}, {-(-Lq // QUERY_BLOCK)}, count], not {tuple(blocks.shape)}"
    dev = nv.require_gpu(q, k, v, blocks, lengths, out)
    lengths = _lengths(lengths, B, dev, Lk)
    if blocks.dtype != torch.int32:
        blocks = blocks.long().clamp(-1, 2 ** 31 - 1).to(torch.int32)
    blocks = blocks.contiguous()
    o = torch.empty(q.shape, dtype=q.dtype, device=dev) if out is None else out
    assert o.shape == q.shape and (o.numel() == 0 or o.stride(3) == 1), f"block_sparse_attention: out is {tuple(q.shape)} with contiguous heads"
    if o.numel() == 0:
        return o
    q, k, v = _bhld_view(q), _bhld_view(k), _bhld_view(v)
    a = nv.SparseAttentionArgs(nv.src4(q), nv.src4(k), nv.src4(v), o.data_ptr(), o.stride(0), o.stride(1), o.stride(2), blocks.data_ptr(), nv.ptr(lengths),
                               B, Hq, Hk, Lq, Lk, blocks.shape[3], D, 1 / math.sqrt(D) if sm_scale is None else float(sm_scale))
    with nv.on_device(dev):
        need = nv.lib().flux_sparse_attention_workspace_bytes(nv.byref(a))
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
        rc = nv.lib().flux_sparse_attention_bf16(nv.byref(a), nv.ptr(ws), need, nv.stream_ptr(dev))
    nv.check(rc, "flux_sparse_attention_bf16")
    return o


def block_sparse_attention(q: Tensor, k: Tensor, v: Tensor, blocks: Tensor, sm_scale: float | None = None, *, lengths: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """Attention of each block of 128 queries over the blocks of 64 keys that its list names, [B, Hq, Lq, D] bf16.

    q, k, v  : bf16 [B, Hq, Lq, D] and [B, Hk, Lk, D] views, heads of 64 or 128; Hq is a multiple of Hk, query head h reads key head h // (Hq // Hk)
    blocks   : whole numbers [B, Hq, ceil(Lq / 128), count], as select_blocks gives them or any others, in any order. A number that is no block of
               the sequence, -1 for one, names nothing, a number that stands there twice counts twice
    sm_scale : factor of the scores, 1 / sqrt(D) if None
    lengths  : whole numbers [B], or None: keys from lengths[b] on are not there
    out      : where the result goes, a [B, Hq, Lq, D] view with contiguous heads, 16-byte aligned rows and memory of its own

    Rows that see no key are 0. Scores and sums are fp32; the probabilities are rounded to bf16 for the matrix cores, as in
    scaled_dot_product_attention. It is not differentiated: a gradient that reaches it raises NotImplementedError.
    """
    if is_dynamo_compiling():
        return torch.compiler.disable(block_sparse_attention)(q, k, v, blocks, sm_scale, lengths=lengths, out=out)
    o = nv.ops().block_sparse_attention(q, k, v, blocks, sm_scale, lengths, out)
    if o is not None:
        return o
    if out is not None:
        assert not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, out))), "block_sparse_attention: a result that goes to `out` is not differentiated"
        if any(unpack_dual(t).tangent is not None for t in (q, k, v, out)):
            raise NotImplementedError("block_sparse_attention has no forward-mode derivative")
        return _launch_sparse(q, k, v, blocks, sm_scale, lengths, out)
    return _block_sparse_attention.apply(q, k, v, blocks, sm_scale, lengths, None)
