"""apply_rope: rotate q and k by per-position 2x2 matrices (kernels/positional_embedding.py:55-82 of
the reference), plus the fused gather flux_qkv_prep it is a special case of. apply_rope_nd, which the reference
does not have, rotates by positions of several axes without such matrices, and rope_table makes them."""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor
from torch.compiler import is_dynamo_compiling

from triton_kernels import _native as nv


def _row_view(t: Tensor) -> Tensor:
    """[B,H,L,D] tensor whose last dim is contiguous and whose strides keep 16-byte addressing."""
    vec = 16 // t.element_size()
    if t.stride(-1) != 1 or any(s % vec for s in t.stride()[:-1]) or t.data_ptr() % 16:
        t = t.contiguous()
    return t


def _pe_table(pe: Tensor, B: int, L: int, D: int) -> tuple[Tensor, int]:
    """fp32 [.., L, D/2, 2, 2] -> contiguous table and its batch stride (0 = shared by all batches).
    The reference kernel reads the first [L, D/2, 2, 2] table whatever the leading extents are
    (kernels/positional_embedding.py:31-32). A head extent is treated the same way here (the first
    head's table serves all heads); a batch extent equal to B is honoured, as broadcasting in the
    plain-PyTorch apply_rope would."""
    assert pe.shape[-4:] == (L, D // 2, 2, 2), f"freqs_cis must end in [{L}, {D // 2}, 2, 2], got {tuple(pe.shape)}"
    if pe.dim() >= 6 and pe.shape[-5] > 1:
        pe = pe.narrow(-5, 0, 1)
    lead = pe.shape[:-4]
    if pe.dtype != torch.float32:
        pe = pe.float()
    pe = pe.contiguous()
    n_lead = 1
    for s in lead:
        n_lead *= s
    if n_lead == 1:
        return pe, 0
    if len(lead) == 2 and lead[0] == B and lead[1] == 1:
        return pe, L * D * 2
    raise NotImplementedError(f"freqs_cis with leading shape {tuple(lead)}: only [1,1,...] or [B,1,...] are supported")


def qkv_prep(q_img: Tensor | None, k_img: Tensor | None, v_img: Tensor | None,
             q_txt: Tensor | None = None, k_txt: Tensor | None = None, v_txt: Tensor | None = None, *,
             pe: Tensor | None = None,
             q_scale_img: Tensor | None = None, k_scale_img: Tensor | None = None,
             q_scale_txt: Tensor | None = None, k_scale_txt: Tensor | None = None,
             eps: float = 1e-6):
    """One streaming pass: concat(txt, img) along the sequence, optional per-head RMS norm of q/k,
    optional RoPE of q/k, v copied. Returns (q, k, v) contiguous [B,H,Lt+Li,D]; entries whose inputs
    were None come back as None. All sources are [B,H,L*,D] views (any batch/head/row strides)."""
    if is_dynamo_compiling():
        return torch.compiler.disable(qkv_prep)(q_img, k_img, v_img, q_txt, k_txt, v_txt, pe=pe, q_scale_img=q_scale_img, k_scale_img=k_scale_img, q_scale_txt=q_scale_txt,
                                                k_scale_txt=k_scale_txt, eps=eps)
    outs = nv.ops().qkv_prep(q_img, k_img, v_img, q_txt, k_txt, v_txt, pe, q_scale_img, k_scale_img, q_scale_txt, k_scale_txt, eps)
    if outs is not None:
        return outs
    ref = next(t for t in (q_img, k_img, v_img) if t is not None)
    B, H, Li, D = ref.shape
    txt_ref = next((t for t in (q_txt, k_txt, v_txt) if t is not None), None)
    Lt = 0 if txt_ref is None else txt_ref.shape[2]
    dev = nv.require_gpu(q_img, k_img, v_img, q_txt, k_txt, v_txt, pe)
    L = Lt + Li
    a = nv.QkvPrepArgs()
    keep = []
    outs = []
    for name, img, txt in (("q", q_img, q_txt), ("k", k_img, k_txt), ("v", v_img, v_txt)):
        if img is None:
            outs.append(None)
            continue
        assert img.shape == (B, H, Li, D) and img.dtype == ref.dtype
        img = _row_view(img)
        keep.append(img)
        setattr(a, f"{name}_img", nv.src4(img))
        if Lt:
            assert txt is not None and txt.shape == (B, H, Lt, D) and txt.dtype == ref.dtype
            txt = _row_view(txt)
            keep.append(txt)
            setattr(a, f"{name}_txt", nv.src4(txt))
        out = torch.empty((B, H, L, D), dtype=ref.dtype, device=dev)
        setattr(a, f"{name}_out", out.data_ptr())
        outs.append(out)
    scales = [q_scale_img, k_scale_img, q_scale_txt, k_scale_txt]
    if any(s is not None for s in scales):
        sdt = next(s for s in scales if s is not None).dtype
        if not (sdt == ref.dtype or (ref.dtype == torch.bfloat16 and sdt == torch.float32)):
            sdt = ref.dtype
        fixed = []
        for s in scales:
            if s is not None:
                assert s.shape[-1] == D
                s = s.to(sdt).contiguous()
                keep.append(s)
            fixed.append(s)
        a.q_scale_img, a.k_scale_img, a.q_scale_txt, a.k_scale_txt = [nv.ptr(s) for s in fixed]
        a.scale_dtype = nv._DTYPE_CODE[sdt]
    else:
        a.scale_dtype = nv.dtype_code(ref)
    if pe is not None:
        table, stride = _pe_table(pe, B, L, D)
        keep.append(table)
        a.pe = table.data_ptr()
        a.pe_batch_stride = stride
    a.B, a.H, a.Lt, a.Li, a.D = B, H, Lt, Li, D
    a.dtype = nv.dtype_code(ref)
    a.eps = float(eps)
    with nv.on_device(dev):
        rc = nv.lib().flux_qkv_prep(nv.byref(a), nv.stream_ptr(dev))
    nv.check(rc, "flux_qkv_prep")
    return tuple(outs)


def apply_rope(xq: Tensor, xk: Tensor, freqs_cis: Tensor) -> tuple[Tensor, Tensor]:
    if is_dynamo_compiling():
        return torch.compiler.disable(apply_rope)(xq, xk, freqs_cis)
    both = nv.ops().apply_rope(xq, xk, freqs_cis)
    if both is not None:
        return both
    assert xq.dim() == 4 and xq.shape == xk.shape and xq.dtype == xk.dtype
    q, k, _ = qkv_prep(xq, xk, None, pe=freqs_cis)
    return q, k


_IDS_DTYPE = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}


def _not_differentiated(ids: Tensor) -> None:
    if torch.is_grad_enabled() and ids.requires_grad:
        raise NotImplementedError("positions are not differentiated")


def _rope_ids(ids: Tensor, axes_dim, theta: float, B: int | None = None, L: int | None = None) -> tuple["nv.RopeIds", Tensor]:
    """The positions as the library takes them, and what has to live until the launch."""
    axes = [int(d) for d in axes_dim]
    assert ids.dim() in (2, 3) and ids.shape[-1] == len(axes), f"ids must be [L, {len(axes)}] or [B, L, {len(axes)}], got {tuple(ids.shape)}"
    assert 1 <= len(axes) <= 8 and all(d > 0 and d % 2 == 0 for d in axes), f"one to eight axes of an even number of values, got {axes}"
    if L is not None:
        assert ids.shape[-2] == L and (ids.dim() == 2 or ids.shape[0] in (1, B)), f"ids of shape {tuple(ids.shape)} for {B} sequences of {L}"
    if ids.dtype not in _IDS_DTYPE:
        if ids.dtype == torch.bool or ids.is_complex():
            raise TypeError(f"unsupported dtype {ids.dtype} of ids")
        ids = ids.float() if ids.is_floating_point() else ids.to(torch.int64)
    sb = ids.stride(0) if ids.dim() == 3 and ids.shape[0] > 1 else 0
    return nv.RopeIds(ids.data_ptr(), sb, ids.stride(-2), ids.stride(-1), float(theta), _IDS_DTYPE[ids.dtype], len(axes), (ctypes.c_int32 * 8)(*axes)), ids


def _rotated(q: Tensor | None, k: Tensor | None, ids: Tensor, axes_dim, theta: float, inverse: bool) -> tuple[Tensor | None, Tensor | None]:
    ref = q if q is not None else k
    B, _, L, D = ref.shape
    dev = nv.require_gpu(q, k, ids)
    at, keep = _rope_ids(ids, axes_dim, theta, B, L)
    outs = []
    a = nv.RopeNdArgs(at=at, B=B, L=L, D=D, dtype=nv.dtype_code(ref), inverse=inverse)
    for name, x in (("q", q), ("k", k)):
        if x is None:
            outs.append(None)
            continue
        if x.stride(3) != 1:
            x = x.contiguous()
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
        setattr(a, name, nv.src4(x))
        setattr(a, f"{name}_out", out.data_ptr())
        setattr(a, f"H{name}", x.shape[1])
        keep = (keep, x)
        outs.append(out)
    with nv.on_device(dev):
        rc = nv.lib().flux_rope_nd(nv.byref(a), nv.stream_ptr(dev))
    nv.check(rc, "flux_rope_nd")
    return tuple(outs)


class _apply_rope_nd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xq, xk, ids, axes_dim, theta):
        ctx.save_for_backward(ids)
        ctx.set_materialize_grads(False)
        ctx.axes_dim, ctx.theta = axes_dim, theta
        return _rotated(xq, xk, ids, axes_dim, theta, False)

    @staticmethod
    def backward(ctx, dq, dk):
        """A rotation's backward pass is the rotation by the negative angles."""
        if dq is None and dk is None:
            return None, None, None, None, None
        ids, = ctx.saved_tensors
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        return (*_apply_rope_nd_inverse.apply(dq, dk, ids, ctx.axes_dim, ctx.theta), None, None, None)


class _apply_rope_nd_inverse(torch.autograd.Function):
    """The backward pass as a function of its own, so that it is differentiable in turn."""

    @staticmethod
    def forward(ctx, dq, dk, ids, axes_dim, theta):
        ctx.save_for_backward(ids)
        ctx.set_materialize_grads(False)
        ctx.axes_dim, ctx.theta = axes_dim, theta
        return _rotated(dq, dk, ids, axes_dim, theta, True)

    @staticmethod
    def backward(ctx, q, k):
        if q is None and k is None:
            return None, None, None, None, None
        ids, = ctx.saved_tensors
        return (*_apply_rope_nd.apply(q, k, ids, ctx.axes_dim, ctx.theta), None, None, None)


def apply_rope_nd(xq: Tensor, xk: Tensor | None, ids: Tensor, axes_dim, theta: float = 10000.0) -> tuple[Tensor, Tensor | None]:
    """q and k rotated by positions of several axes (time, height, width), with gradients for both.

    xq, xk : [B, H, L, D] views with any strides, B 65535 at most; xk may have another number of heads or be None. bf16 or fp32.
    ids : the tokens' positions, [B, L, n] or [L, n] for all batch elements: float32, float64, int32 or int64 (others are converted).
    axes_dim : values of a row that belong to each of the n axes, in order; even, D in all, at most 512.
    Pair j of an axis of d values turns by ids[b, l, axis] * theta^(-2j/d), formed in 64 bits: apply_rope with EmbedND's table, without the
    table. The results are contiguous and rounded once.
    """
    if is_dynamo_compiling():
        return torch.compiler.disable(apply_rope_nd)(xq, xk, ids, axes_dim, theta)
    both = nv.ops().apply_rope_nd(xq, xk, ids, axes_dim, theta)
    if both is not None:
        return both
    for x in (xq, xk):
        assert x is None or (x.dim() == 4 and x.dtype == xq.dtype), "q and k are [B, H, L, D] of one type"
    B, _, L, D = xq.shape
    assert xk is None or (xk.shape[0], *xk.shape[2:]) == (B, L, D), f"q {tuple(xq.shape)} and k {tuple(xk.shape)} differ in more than their heads"
    axes = tuple(int(d) for d in axes_dim)
    assert sum(axes) == D, f"axes of {sum(axes)} values in all for rows of {D}"
    _not_differentiated(ids)
    return _apply_rope_nd.apply(xq, xk, ids, axes, float(theta))


def rope_table(ids: Tensor, axes_dim, theta: float = 10000.0) -> Tensor:
    """The fp32 rotation matrices that the blocks and apply_rope take, [B, 1, L, D/2, 2, 2] for ids [B, L, n] ([1, 1, ...] for [L, n]):
    one kernel for what EmbedND of the plain blocks computes; arguments as in apply_rope_nd."""
    if is_dynamo_compiling():
        return torch.compiler.disable(rope_table)(ids, axes_dim, theta)
    out = nv.ops().rope_table(ids, axes_dim, theta)
    if out is not None:
        return out
    dev = nv.require_gpu(ids)
    _not_differentiated(ids)
    at, _keep = _rope_ids(ids, axes_dim, theta)
    B, L = ids.shape[0] if ids.dim() == 3 else 1, ids.shape[-2]
    out = torch.empty((B, 1, L, sum(at.axes_dim) // 2, 2, 2), dtype=torch.float32, device=dev)
    with nv.on_device(dev):
        rc = nv.lib().flux_rope_table(nv.byref(at), out.data_ptr(), B, L, nv.stream_ptr(dev))
    nv.check(rc, "flux_rope_table")
    return out
