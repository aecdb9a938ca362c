"""layer_norm of rows beyond the registers (and just below), with rows and gradients in every order; bounds of test_layer_norm."""
import pytest
import torch

import triton_kernels as tk
from test_layer_norm import check, inputs
from util import DEV, randn, seeded


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [16384, 16392, 16401, 40000])
def test_strides(n, dtype):
    g = seeded(n)
    base = randn(g, 3, 5, 2, n + 8, dtype=dtype).to(DEV)
    w, b = randn(g, 3, 1, n, dtype=dtype).to(DEV), randn(g, n, dtype=dtype).to(DEV)
    x, dy = base[:, :, 0, :n], base[:, :, 1, 8:]
    check(x, w, b, dy)                                                                # rows two apart, dy of other strides
    check(x, b, w, base[:1, :1, 1, :n].expand(3, 5, n), plus_one=True)                # an expanded gradient
    check(x, w, b, randn(g, 3, n, 5, dtype=dtype).to(DEV).transpose(1, 2))            # last dimension strided
    check(base[:, :1, 0, 1:n + 1].expand(3, 5, n), b, None, dy, wanted="xw")          # the same row, at odd addresses
    check(x.transpose(0, 1), b, b, dy.transpose(0, 1), wanted="wb")
    check(x[0, 0], b, b, dy[0, 0])                                                    # one row
    leaf = x.detach().clone().requires_grad_(True)
    dx, = torch.autograd.grad(tk.layer_norm(leaf, w, b).sum(), leaf)                  # (sum's gradient: one value, expanded over all dimensions)
    want, = torch.autograd.grad(tk.layer_norm(leaf, w, b), leaf, torch.ones_like(leaf))
    assert torch.equal(dx, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(300, 16392), (129, 33000)])
def test_many_rows(rows, n):
    (x, dy), g = inputs((rows, n), torch.bfloat16, n)
    check(x, randn(g, n).to(DEV), randn(g, n).to(DEV), dy)
