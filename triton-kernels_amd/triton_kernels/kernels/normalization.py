"""rms_norm, layer_norm_modulation and layer_norm: Python launchers over the HIP row-wise kernels.

Same call signatures, defaults and assertion behaviour as kernels/normalization.py:47-77 and
:142-193 of the reference; the device work is flux_rms_norm / flux_rms_norm_bwd /
flux_layer_norm_modulation in libfluxhip.so. layer_norm, which the reference does not have, is the layer norm
that can be trained (flux_layer_norm / flux_layer_norm_bwd).
"""
from __future__ import annotations

import torch
from torch.compiler import is_dynamo_compiling

from triton_kernels import _native as nv
from triton_kernels.kernels.utils import calculate_settings


def _as_4d_view(x: torch.Tensor):
    """Sizes (d0,d1,d2) and strides (s0,s1,s2) of x seen as [d0,d1,d2,n] rows, without copying when x
    has at most four dims and a contiguous last dim; otherwise a contiguous copy is described."""
    if x.dim() == 0:
        raise AssertionError("rms_norm needs at least one dimension")
    if x.dim() > 4 or x.stride(-1) != 1:
        x = x.contiguous()
        if x.dim() > 4:
            x = x.reshape(-1, x.shape[-1])
    lead, strides = tuple(x.shape)[:-1], x.stride()[:-1]
    short = 3 - len(lead)
    if short:
        lead, strides = (1,) * short + lead, (0,) * short + strides
    return x, lead, strides


def _rms_norm_args(x: torch.Tensor, scale: torch.Tensor, want_rstd: bool = False):
    """The call's arguments in the order of nv.RmsNormArgs, its outputs and the tensors that have to live until
    it is launched."""
    shape, dtype = x.shape, x.dtype
    assert shape[-1] == scale.shape[-1]
    dev = nv.require_gpu(x, scale)
    if shape[-1] > nv.MAX_ROW:
        calculate_settings(shape[-1])  # raises, like the reference
    scale = scale.contiguous()
    if scale.dtype != dtype and not (dtype == torch.bfloat16 and scale.dtype == torch.float32):
        scale = scale.to(dtype)
    xv, lead, strides = _as_4d_view(x)
    y = torch.empty(shape, dtype=dtype, device=dev)
    rstd = torch.empty((lead[0] * lead[1] * lead[2],), dtype=torch.float32, device=dev) if want_rstd else None
    return (xv.data_ptr(), scale.data_ptr(), y.data_ptr(), rstd.data_ptr() if want_rstd else None, *lead, *strides), y, rstd, (xv, scale)


def rms_norm_forward(x: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6, want_rstd: bool = False):
    a, y, rstd, (xv, scale) = _rms_norm_args(x, scale, want_rstd)
    dev = y.device
    with nv.on_device(dev):
        rc = nv.lib().flux_rms_norm(
            *a[:7], y.shape[-1], *a[7:],
            nv.dtype_code(y), nv.dtype_code(scale), float(eps), nv.stream_ptr(dev))
    nv.check(rc, "flux_rms_norm")
    return y, rstd, xv


def _vector_rows(x: torch.Tensor) -> bool:
    """Whether every row of x starts on a 16-byte boundary, where the kernel holds a row in registers."""
    per16 = 16 // x.element_size()
    return x.data_ptr() % 16 == 0 and x.shape[-1] % per16 == 0 and all(s % per16 == 0 for s in x.stride()[:-1])


class _rms_norm(torch.autograd.Function):
    """y = x * rsqrt(mean(x^2, -1) + eps) * scale with a HIP forward and backward.

    grad_mode = False says that nothing will be differentiated (a parameter's requires_grad stays true under
    no_grad): a view with 16-byte rows is then read in place and no rstd is kept. Rows that are not 16-byte
    addressable are still copied first, since the kernel for such rows reads a row twice by elements."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6, grad_mode: bool = True) -> torch.Tensor:
        need_grad = x.requires_grad or scale.requires_grad
        if need_grad and (grad_mode or not _vector_rows(x)):
            x = x.contiguous()
        need_grad = need_grad and grad_mode
        y, rstd, _ = rms_norm_forward(x, scale, eps, want_rstd=need_grad)
        if need_grad:
            ctx.save_for_backward(x.reshape(-1, x.shape[-1]), scale.contiguous(), rstd)
        return y

    @staticmethod
    def backward(ctx, dy: torch.Tensor):
        x2, scale, rstd = ctx.saved_tensors   # (what saved-tensor hooks gave back, of any type)
        dev = nv.require_gpu(dy, x2, scale, rstd)
        rows, n = x2.shape
        if scale.numel() != n or rstd.numel() != rows:
            raise RuntimeError("rms_norm: saved tensors came back with other sizes")
        x2, rstd = x2.contiguous(), rstd.float().contiguous()
        dy2 = dy.contiguous().reshape(rows, n)
        if dy2.dtype != x2.dtype:
            dy2 = dy2.to(x2.dtype)
        sc = scale.contiguous()
        if sc.dtype != x2.dtype and not (x2.dtype == torch.bfloat16 and sc.dtype == torch.float32):
            sc = sc.to(x2.dtype)
        dx = torch.empty_like(x2)
        # the kernel's types; the gradient of a scale of another type is converted from fp32 below
        dscale = torch.empty((n,), dtype=scale.dtype if scale.dtype == torch.bfloat16 else torch.float32, device=dev)
        xcode = nv.dtype_code(x2)
        ws = torch.empty((nv.lib().flux_rms_norm_bwd_workspace_bytes(rows, n, xcode),), dtype=torch.uint8, device=dev)
        with nv.on_device(dev):
            rc = nv.lib().flux_rms_norm_bwd_ws(
                dy2.data_ptr(), x2.data_ptr(), sc.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dscale.data_ptr(), nv.dtype_code(dscale),
                ws.data_ptr(), ws.numel(), rows, n, xcode, nv.dtype_code(sc), nv.stream_ptr(dev))
        nv.check(rc, "flux_rms_norm_bwd")
        return dx.reshape(dy.shape), dscale.to(scale.dtype).reshape(scale.shape), None, None


def rms_norm(x: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    if is_dynamo_compiling():
        return torch.compiler.disable(rms_norm)(x, scale, eps)
    y = nv.ops().rms_norm(x, scale, eps)
    return _rms_norm.apply(x, scale, eps, torch.is_grad_enabled()) if y is None else y


class _rms_norm_pair(torch.autograd.Function):
    """rms_norm of two tensors in one launch, for calls that are not differentiated. A Function all the same, so
    that forward-mode derivatives and function transforms are refused as they are by rms_norm."""

    @staticmethod
    def forward(ctx, x0, scale0, x1, scale1, eps):
        a0, y0, _, (_x0, s0) = _rms_norm_args(x0, scale0)
        a1, y1, _, (_x1, s1) = _rms_norm_args(x1, scale1)
        dev = y0.device
        with nv.on_device(dev):
            rc = nv.lib().flux_rms_norm_pair(
                nv.byref(nv.RmsNormArgs(*a0)), nv.byref(nv.RmsNormArgs(*a1)), y0.shape[-1], nv.dtype_code(y0), nv.dtype_code(s0), float(eps), nv.stream_ptr(dev))
        nv.check(rc, "flux_rms_norm_pair")
        return y0, y1


def rms_norm_pair(x0, scale0, x1, scale1, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(rms_norm(x0, scale0), rms_norm(x1, scale1)): one launch where nothing is differentiated and the two have
    the same width, types and device and 16-byte rows, two calls otherwise. At [1, 24, 256, 128] (q and k of one projection) the
    two calls took 50 us of host time, the copies of the views included; this takes 23, and 8 in native code."""
    if is_dynamo_compiling():
        return torch.compiler.disable(rms_norm_pair)(x0, scale0, x1, scale1, eps)
    y = nv.ops().rms_norm_pair(x0, scale0, x1, scale1, eps)
    if y is not None:
        return y
    if (torch.is_grad_enabled() or x0.dtype != x1.dtype or x0.device != x1.device or scale0.dtype != scale1.dtype
            or not x0.dim() or not x1.dim() or x0.shape[-1] != x1.shape[-1] or not (_vector_rows(x0) and _vector_rows(x1))):
        return rms_norm(x0, scale0, eps), rms_norm(x1, scale1, eps)
    return _rms_norm_pair.apply(x0, scale0, x1, scale1, eps)


def layer_norm_modulation(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps=1e-5) -> torch.Tensor:
    """(1 + weight) * layer_norm(x) + bias, where weight is the adaLN *scale* and bias the *shift*,
    each [B, 1, N] (or [B, N]); chunks of a wider modulation tensor are read in place."""
    if is_dynamo_compiling():
        return torch.compiler.disable(layer_norm_modulation)(x, weight, bias, eps)
    y = nv.ops().layer_norm_modulation(x, weight, bias, eps)
    if y is not None:
        return y
    a, y, _keep = _layer_norm_args(x, weight, bias)
    dev = y.device
    with nv.on_device(dev):
        rc = nv.lib().flux_layer_norm_modulation(
            *a[:6], y.shape[-1], a[6], nv.dtype_code(y), float(eps), nv.stream_ptr(dev))
    nv.check(rc, "flux_layer_norm_modulation")
    return y


def layer_norm_modulation_pair(first: tuple, second: tuple, eps=1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """layer_norm_modulation of two (x, weight, bias) triples of the same width and type in one launch."""
    if is_dynamo_compiling():
        return torch.compiler.disable(layer_norm_modulation_pair)(first, second, eps)
    y = nv.ops().layer_norm_modulation_pair(*first, *second, eps) if len(first) == len(second) == 3 else None
    if y is not None:
        return y
    a0, y0, _keep0 = _layer_norm_args(*first)
    a1, y1, _keep1 = _layer_norm_args(*second)
    assert y0.shape[-1] == y1.shape[-1] and y0.dtype == y1.dtype and y0.device == y1.device
    dev = y0.device
    with nv.on_device(dev):
        rc = nv.lib().flux_layer_norm_modulation_pair(
            nv.byref(nv.LayerNormArgs(*a0)), nv.byref(nv.LayerNormArgs(*a1)), y0.shape[-1], nv.dtype_code(y0), float(eps), nv.stream_ptr(dev))
    nv.check(rc, "flux_layer_norm_modulation_pair")
    return y0, y1


def _layer_norm_args(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor):
    """The call's arguments in the order of nv.LayerNormArgs, its output and the tensors that have to live until
    it is launched."""
    shape, weight_shape, bias_shape = x.shape, weight.shape, bias.shape
    batch, n = shape[0], shape[-1]
    assert batch == weight_shape[0] == bias_shape[0]
    assert n == weight_shape[-1] == bias_shape[-1]
    nv.require_gpu(x, weight, bias)
    if n > nv.MAX_ROW:
        calculate_settings(n)
    x = x.contiguous()
    if weight.dtype != x.dtype:
        weight = weight.to(x.dtype)
    if bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    assert weight.numel() == batch * n and bias.numel() == batch * n, "scale/shift must be [B, 1, N]"
    in_place = weight.stride(-1) == 1 and bias.stride(-1) == 1 and (batch == 1 or weight.stride(0) == bias.stride(0))
    if not in_place:
        weight, bias = weight.contiguous(), bias.contiguous()
    mod_stride = weight.stride(0) if batch > 1 else n
    if batch > 1 and mod_stride < n:
        weight, bias = weight.contiguous(), bias.contiguous()
        mod_stride = weight.stride(0)
    y = torch.empty_like(x)
    rows = x.numel() // n
    return (x.data_ptr(), weight.data_ptr(), bias.data_ptr(), y.data_ptr(), batch, rows // batch if batch else 0, mod_stride), y, (x, weight, bias)


class _layer_norm(torch.autograd.Function):
    """layer_norm of an x seen as [batch, seq, n], with weight and bias [groups, n] (or None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, plus_one, grad_mode):
        batch, seq, n = x.shape
        dev = x.device
        need_grad = grad_mode and any(ctx.needs_input_grad[:3])
        y = torch.empty((batch, seq, n), dtype=x.dtype, device=dev)
        stats = torch.empty((2, batch * seq), dtype=torch.float32, device=dev) if need_grad else (None, None)
        a = nv.LayerNormFwdArgs(x.data_ptr(), nv.ptr(weight), nv.ptr(bias), y.data_ptr(), nv.ptr(stats[0]), nv.ptr(stats[1]),
                                batch, seq, x.stride(0), x.stride(1), groups, weight.stride(0) if weight is not None else 0, bias.stride(0) if bias is not None else 0,
                                n, nv.dtype_code(x), nv.dtype_code(x if weight is None and bias is None else weight if weight is not None else bias), plus_one, eps)
        if batch * seq:
            with nv.on_device(dev):
                rc = nv.lib().flux_layer_norm(nv.byref(a), nv.stream_ptr(dev))
            nv.check(rc, "flux_layer_norm")
        if need_grad:
            ctx.save_for_backward(x, weight, stats)
            ctx.groups, ctx.plus_one, ctx.bias_dtype = groups, plus_one, None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors   # (what saved-tensor hooks gave back)
        return (*_layer_norm_grads.apply(dy, x, weight, stats, ctx.groups, ctx.plus_one, ctx.bias_dtype, ctx.needs_input_grad[:3]), None, None, None, None)


class _layer_norm_grads(torch.autograd.Function):
    """Its gradients. A Function, so that what they depend on has an edge to an error where they are recorded (create_graph), not to nothing."""

    @staticmethod
    def forward(ctx, dy, x, weight, stats, groups, plus_one, bias_dtype, wanted):
        want_x, want_w, want_b = wanted
        dev = nv.require_gpu(dy, x, weight, stats)
        batch, seq, n = dy.shape
        if x.shape != dy.shape or stats.shape != (2, batch * seq) or (weight is not None and weight.shape != (groups, n)):
            raise RuntimeError("layer_norm: saved tensors came back with other sizes")
        x, dy = _unit_stride(x), _unit_stride(dy if dy.dtype == x.dtype else dy.to(x.dtype))
        stats = stats.float().contiguous()
        w_dtype = weight.dtype if weight is not None else bias_dtype or x.dtype
        if weight is not None:
            weight = _unit_stride(weight)
        dx = torch.empty((batch, seq, n), dtype=x.dtype, device=dev) if want_x else None
        sums = torch.empty if batch * seq else torch.zeros
        dw = sums((groups, n), dtype=w_dtype, device=dev) if want_w else None
        db = sums((groups, n), dtype=w_dtype, device=dev) if want_b else None
        if batch * seq:
            a = nv.LayerNormBwdArgs(dy.data_ptr(), x.data_ptr(), nv.ptr(weight), stats[0].data_ptr(), stats[1].data_ptr(), nv.ptr(dx), nv.ptr(dw), nv.ptr(db),
                                    batch, seq, dy.stride(0), dy.stride(1), x.stride(0), x.stride(1), groups, weight.stride(0) if weight is not None else 0,
                                    n, nv.dtype_code(x), nv._DTYPE_CODE[w_dtype], plus_one)
            need = nv.lib().flux_layer_norm_bwd_workspace_bytes(nv.byref(a))
            ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
            with nv.on_device(dev):
                rc = nv.lib().flux_layer_norm_bwd(nv.byref(a), nv.ptr(ws), need, nv.stream_ptr(dev))
            nv.check(rc, "flux_layer_norm_bwd")
        return dx, dw, db

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("layer_norm is differentiated once only")


def _unit_stride(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5, *, plus_one: bool = False) -> torch.Tensor:
    """layer_norm(x) * weight + bias over the last dimension, with gradients for all three; rounded once.

    weight, bias : [N], shared by all rows, or one for each element of x's first dimension, [B, N] or [B, 1, ..., N] (chunks of a wider modulation
    tensor are read in place), 65535 of them at most; either may be None. Their gradients are sums over the rows that share them, formed in fp32.
    plus_one : the factor is 1 + weight, adaLN's scale. layer_norm_modulation is that operator for inference, in the rounding order of
    PyTorch's bf16 operations and without gradients.
    x is bf16 or fp32, [..., N] with N up to 65536. weight and bias may be of other types than x, and each of its own: unless both are of x's they are taken
    as fp32, and their gradients come in their types.
    """
    if is_dynamo_compiling():
        return torch.compiler.disable(layer_norm)(x, weight, bias, eps, plus_one=plus_one)
    y = nv.ops().layer_norm(x, weight, bias, eps, plus_one)
    if y is not None:
        return y
    nv.require_gpu(x, weight, bias)
    assert x.dim() >= 1, "layer_norm needs at least one dimension"
    nv.dtype_code(x)
    n = x.shape[-1]
    if n > nv.MAX_ROW:
        calculate_settings(n)
    batch = x.shape[0] if x.dim() > 1 else 1
    per_batch = False
    for t in (weight, bias):
        if t is None:
            continue
        assert t.dim() >= 1 and t.shape[-1] == n, f"weight and bias are [{n}] or one such vector for each of {batch} batch elements, not {tuple(t.shape)}"
        if t.numel() != n:
            assert x.dim() > 1 and t.dim() > 1 and t.shape[0] == batch and t.numel() == batch * n, \
                f"weight and bias are [{n}] or one such vector for each of {batch} batch elements, not {tuple(t.shape)}"
            per_batch = True
    groups = batch if per_batch else 1

    def vectors(t, dtype):
        if t is None:
            return None
        if t.dtype != dtype:
            t = t.to(dtype)
        t = t.reshape(1 if t.numel() == n else groups, n)
        return _unit_stride(t if t.shape[0] == groups else t.expand(groups, n))

    # fp32 where either holds more than x's type, and where one of the two is shared: its gradient is the sum of the groups', which are not rounded before that
    w_dtype = x.dtype if all(t is None or t.dtype == x.dtype for t in (weight, bias)) else torch.float32
    if groups > 1 and any(t is not None and t.numel() == n for t in (weight, bias)):
        w_dtype = torch.float32
    rows = _unit_stride(x.reshape(batch, -1, n)) if x.numel() else x.reshape(batch, x.numel() // max(1, batch * n), n)
    y = _layer_norm.apply(rows, vectors(weight, w_dtype), vectors(bias, w_dtype), groups, float(eps), bool(plus_one), torch.is_grad_enabled())
    return y.reshape(x.shape)
