"""layer_norm, apply_rope_nd and linear_lora beyond 2^31 values: what lies behind them against the same rows by themselves."""
import pytest
import torch

import triton_kernels as tk
from util import DEV, randn, seeded

BF = torch.bfloat16


def repeated(g, rows, n):
    """[rows, n] of values that repeat every 1009 rows, so that rows far behind differ from those 2^31 or 2^32 bytes in front of them."""
    return randn(g, 1009, n, dtype=BF).to(DEV).repeat(-(-rows // 1009), 1)[:rows]


@pytest.mark.gpu
def test_layer_norm():
    g = seeded(1)
    n, rows = 3072, 2 ** 31 // 3072 + 999
    x, dy = repeated(g, rows, n).view(1, rows, n).requires_grad_(True), repeated(g, rows, n).view(1, rows, n)
    w, b = randn(g, n, dtype=BF).to(DEV).requires_grad_(True), randn(g, n, dtype=BF).to(DEV).requires_grad_(True)
    y = tk.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    for at in (slice(0, 50), slice(rows - 300, rows)):
        xs = x[:, at].detach().requires_grad_(True)
        ys = tk.layer_norm(xs, w.detach(), b.detach())
        assert torch.equal(ys, y[:, at]) and torch.equal(torch.autograd.grad(ys, xs, dy[:, at])[0], dx[:, at])
    # sums of whole periods and a rest, in 64 bits; 2^-24 times the rows of a chain (2732 of a block) and those of the parts, and one rounding
    part, rest = rows // 1009, rows % 1009
    d = dy[0, :1009].double()
    h = x.detach()[0, :1009].double()
    h = (h - h.mean(-1, keepdim=True)) / torch.sqrt(h.var(-1, correction=0, keepdim=True) + 1e-5)
    for got, terms in ((dw, d * h), (db, d)):
        want = part * terms.sum(0) + terms[:rest].sum(0)
        size = part * terms.abs().sum(0) + terms[:rest].abs().sum(0)
        assert ((got.double() - want).abs() <= (3500 + 512) * 2.0 ** -24 * size + 2.0 ** -8 * want.abs()).all()


@pytest.mark.gpu
def test_apply_rope_nd():
    g = seeded(2)
    H, D = 24, 128
    L = 2 ** 31 // (H * D) + 777
    q = repeated(g, L, H * D).view(1, L, H, D).transpose(1, 2)
    ids = torch.stack((torch.arange(L, device=DEV), torch.arange(L, device=DEV) % 97, torch.arange(L, device=DEV) % 61), -1)
    yq, yk = tk.apply_rope_nd(q, q[:, 20:], ids, (16, 56, 56))
    for at in (slice(0, 40), slice(L - 500, L)):
        one, two = tk.apply_rope_nd(q[:, :, at], q[:, 20:, at], ids[at], (16, 56, 56))
        assert torch.equal(one, yq[:, :, at]) and torch.equal(two, yk[:, :, at])


@pytest.mark.gpu
def test_linear_lora():
    import test_linear_lora
    g, _, w, b, lora_a, lora_b, scaling = test_linear_lora.make(3, (1,), 2056, 2056, 5, 16)
    M = 2 ** 31 // 2056 + 5001
    x, adapter = repeated(g, M, 2056), torch.arange(M, device=DEV) // 700 % 6 - 1
    y = tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling)
    for at in (slice(0, 300), slice(M - 2000, M)):
        want, off = test_linear_lora.exact(x[at], w, b, lora_a, lora_b, adapter[at], scaling, False)
        assert ((y[at].double() - want).abs() <= off + 2.0 ** -8 * want.abs()).all()
