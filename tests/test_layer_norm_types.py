"""layer_norm with a weight and a bias of types of their own: neither is rounded on the way in, nor its gradient on the way out beyond its own type.

Tolerances. u = 2^-24. Inputs of +-1 in equal numbers have mean 0 and h = +-1 within 2^-17 (eps 1e-5 of the variance, 16 u of the sums); the result is h w + b with
a few u of its terms, rounded to bf16 once. A sum of R terms is off by R u of their magnitudes and half a step of its type."""
import pytest
import torch

import triton_kernels as tk
from util import DEV, randn, seeded

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
U = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("w_dtype,b_dtype", [(BF, F32), (F32, BF), (F16, BF), (BF, F16), (F16, F16), (F64, F64), (BF, F64), (F32, F16), (None, F16), (F16, None), (BF, BF), (F32, F32)])
@pytest.mark.parametrize("each", [False, True])
def test_types_of_weight_and_bias(each, w_dtype, b_dtype):
    g = seeded(3)
    B, L, N = 3, 37, 192
    sign = torch.cat((torch.ones(N // 2), -torch.ones(N // 2)))
    x = torch.stack([sign[torch.randperm(N, generator=g)] for _ in range(B * L)]).view(B, L, N).to(DEV, BF).requires_grad_(True)
    shape = (B, 1, N) if each else (N,)
    # what the types hold beyond bf16's eight bits, so that w and b nearly cancel in half of the values
    fine = 2.0 ** -9 * torch.rand(shape, generator=g) + 2.0 ** -10
    w = None if w_dtype is None else (1 + fine).to(DEV, w_dtype).requires_grad_(True)
    b = None if b_dtype is None else (-1 + fine).to(DEV, b_dtype).requires_grad_(True)
    dy = randn(g, B, L, N, dtype=BF).to(DEV)
    y = tk.layer_norm(x, w, b)
    xd = x.detach().double()
    h = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-5)
    f, s = (1.0 if w is None else w.detach().double()), (0.0 if b is None else b.detach().double())
    want = h * f + s
    assert y.dtype == BF and ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * U).all(), (y.double() - want).abs().max()
    leaves = [t for t in (x, w, b) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy))
    assert [t.dtype for t in grads] == [t.dtype for t in leaves]
    over, d = (1 if each else (0, 1)), dy.double()
    for leaf, got, terms in ((w, None, d * h), (b, None, d)):
        if leaf is None:
            continue
        got = grads[1] if leaf is w else grads[-1]
        ref, size = terms.sum(over).view(shape), terms.abs().sum(over).view(shape)
        half = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: U, F64: U}[leaf.dtype]   # (fp64's goes through fp32)
        assert ((got.double() - ref).abs() <= half * ref.abs() + (B * L + 64) * U * size + 2.0 ** -24).all(), (got.double() - ref).abs().max()
