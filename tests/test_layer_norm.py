"""layer_norm, forward and backward, against the formulas in 64 bits.

Tolerances. u = 2^-24. A row's sums are trees of at most 8 x 8 values in a lane, 6 steps in a wave and 16 waves, so mean and variance carry at
most 90 u of the sums of the magnitudes; with |mean| <= 2 std in these inputs h is off by less than H = 512 u (1 + |h|). A result that
is rounded to bf16 adds 2^-8 of its value. A sum over rows adds up at most rows / blocks + 64 + 40 values in a chain, each with its own error."""
import math

import pytest
import torch

import triton_kernels as tk
from util import DEV, randn, seeded

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def half_step(t):
    return {BF: 2.0 ** -8, F32: U}[t]


def exact(x, w, b, dy, eps, plus_one):
    """y, dx, dw, db in 64 bits and how far each may be off; w and b broadcast against x."""
    xd, d = x.double(), dy.double()
    n = x.shape[-1]
    var, mean = torch.var_mean(xd, -1, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = (xd - mean) * rstd
    f = torch.ones_like(xd) if w is None else (w.double() + (1.0 if plus_one else 0.0)).expand_as(xd)
    bias = torch.zeros_like(xd) if b is None else b.double().expand_as(xd)
    H = 512 * U * (1 + h.abs())
    y, y_off = h * f + bias, H * f.abs() + 4 * U * ((h * f).abs() + bias.abs())
    g = d * f
    ga, gh = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    dx_off = 512 * U * rstd * (g.abs() + ga + (1 + h.abs()) * (gh + ga))
    return y, y_off, dx, dx_off, d * h, d.abs() * H, d, n


def summed(t, like):
    """t summed over what `like`, which broadcasts against it, shares."""
    lead = (1,) * (t.dim() - like.dim()) + tuple(like.shape)
    return t.sum([i for i in range(t.dim()) if lead[i] == 1], keepdim=True).reshape(like.shape) if any(s == 1 for s in lead[:-1]) else t.reshape(like.shape)


def check(x, w, b, dy, eps=1e-5, plus_one=False, wanted="xwb"):
    leaves = [t.detach().requires_grad_(name in wanted) if t is not None else None for name, t in (("x", x), ("w", w), ("b", b))]
    y = tk.layer_norm(*leaves, eps, plus_one=plus_one)
    assert y.shape == x.shape and y.dtype == x.dtype
    with torch.no_grad():
        assert torch.equal(tk.layer_norm(x, w, b, eps, plus_one=plus_one), y)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None and t.requires_grad], dy)
    want, y_off, dx, dx_off, dw, dw_off, db, n = exact(x, w, b, dy, eps, plus_one)
    assert ((y.double() - want).abs() <= y_off + half_step(y.dtype) * want.abs()).all(), (y.double() - want).abs().max()
    grads = iter(grads)
    if "x" in wanted:
        got = next(grads)
        assert got.shape == x.shape and got.dtype == x.dtype
        assert ((got.double() - dx).abs() <= dx_off + half_step(x.dtype) * dx.abs()).all(), (got.double() - dx).abs().max()
    chain = (x.numel() // n / 256 + 104) * U
    for name, t, terms, off in (("w", w, dw, dw_off), ("b", b, db, torch.zeros_like(db))):
        if t is None or name not in wanted:
            continue
        got = next(grads)
        assert got.shape == t.shape and got.dtype == t.dtype
        want = summed(terms, t)
        bound = summed(off + chain * terms.abs(), t) + half_step(t.dtype) * want.abs()
        assert ((got.double() - want).abs() <= bound).all(), (name, (got.double() - want).abs().max())


def inputs(shape, dtype, seed):
    g = seeded(seed)
    return [(randn(g, *shape) * (0.5 + torch.rand(shape[-1], generator=g)) + 0.5).to(dtype).to(DEV), randn(g, *shape, dtype=dtype).to(DEV)], g


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype,w_dtype", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("rows,n", [(1, 1), (5, 2), (3, 8), (77, 768), (1, 1024), (2049, 96), (300, 1000), (130, 1001), (9, 2047),   # lanes of one wave, one or more units a lane
                                    (64, 1536), (40, 3000), (1100, 4096), (33, 8200), (7, 12296), (5, 16384),                       # several waves a row
                                    (3, 8193), (6, 16392), (2, 65536), (70, 9001)])                                                 # beyond the registers
def test_shapes(rows, n, x_dtype, w_dtype):
    (x, dy), g = inputs((rows, n), x_dtype, rows + n)
    check(x, randn(g, n, dtype=w_dtype).to(DEV), randn(g, n, dtype=w_dtype).to(DEV), dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("batch,tokens,n", [(1, 1, 64), (3, 1, 1000), (3, 130, 512), (2, 700, 1536), (5, 33, 77), (4, 9, 16400)])
def test_a_weight_for_each_batch_element(batch, tokens, n, dtype):
    (x, dy), g = inputs((batch, tokens, n), dtype, batch + tokens + n)
    shift, scale, _ = (randn(g, batch, 1, 3 * n, dtype=dtype, std=0.3).to(DEV)).chunk(3, -1)     # chunks of a wider tensor
    check(x, scale, shift, dy, 1e-6, True)
    check(x, scale.squeeze(1)[:, None], None, dy, 1e-6, False)
    check(x, None, shift, dy)
    check(x, scale[:1, 0, :].reshape(n).contiguous(), shift, dy)                                  # a shared weight beside a shift of every element
    check(x, scale.mean(0, keepdim=True), shift, dy, plus_one=True)
    check(x, None, None, dy, wanted="x")
    for wanted in ("x", "w", "b", "wb"):
        check(x, scale, shift, dy, 1e-6, True, wanted)


@pytest.mark.gpu
def test_broadcast_weights_get_the_sum_of_their_gradients():
    (x, dy), g = inputs((3, 20, 256), F32, 5)
    one = randn(g, 256).to(DEV).requires_grad_(True)
    wide = one[None, None].expand(3, 1, 256)
    check(x, wide.detach(), None, dy)
    a, = torch.autograd.grad(tk.layer_norm(x, wide), one, dy)
    b, = torch.autograd.grad(tk.layer_norm(x, one), one, dy)
    torch.testing.assert_close(a, b, atol=4e-5, rtol=0)    # 60 terms of size 1 to 10 in two orders: 60 * 10 * 2^-24 = 4e-5 at worst


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_alignment(dtype):
    g = seeded(3)
    base = randn(g, 3, 50, 2, 264, dtype=dtype).to(DEV)
    w, b = randn(g, 264, dtype=dtype).to(DEV), randn(g, 264, dtype=dtype).to(DEV)
    dy = randn(g, 3, 264, 50, dtype=dtype).to(DEV).transpose(1, 2)                     # last dimension strided
    check(base[:, :, 1], w, b, dy)                                                     # rows 2 * 264 apart
    check(base[:, 7:40, 0], w, b, dy[:, :33].contiguous())                             # a slice of a longer sequence
    check(base[:, :, 0].transpose(0, 1), w, b, dy.transpose(0, 1))
    check(base.reshape(3, 50, 4, 132)[..., 1:128], w[1:128], b[:127], base.reshape(3, 50, 4, 132)[..., 2:129])   # odd addresses, 4-d
    check(base[0, 0, 0], w, b, base[1, 0, 0])                                          # one row
    check(base[:, :1, 0].expand(3, 50, 264), w, b, dy)                                 # the same row fifty times
    check(base[:, :, 0], w, b, base[:1, :1, 1].expand(3, 50, 264))                     # an expanded gradient
    odd = torch.empty(3 * 50 * 264 + 1, dtype=dtype, device=DEV)[1:].view(3, 50, 264).copy_(base[:, :, 0])
    check(odd, w, b, dy)                                                               # a base that is not 16-byte aligned


@pytest.mark.gpu
def test_rows_of_their_own():
    """What is not finite in a row stays there; a constant row is all bias; no rows: no values and gradients of zero."""
    (x, dy), g = inputs((2, 64, 512), F32, 9)
    w, b = randn(g, 512).to(DEV), randn(g, 512).to(DEV)
    bad, bad_dy = x.clone(), dy.clone()
    bad[0, 3, 7], bad[1, 0, 0], bad_dy[1, 5, 1] = float("nan"), float("inf"), float("nan")
    bad[0, 9] = 3.0
    bad.requires_grad_(True)
    y = tk.layer_norm(bad, w, b)
    dx, = torch.autograd.grad(y, bad, bad_dy)
    rows = torch.ones(2, 64, dtype=torch.bool, device=DEV)
    rows[0, 3] = rows[1, 0] = False
    assert torch.equal(y.isfinite().all(-1), rows)
    rows[1, 5] = False
    assert torch.equal(dx.isfinite().all(-1), rows)
    assert torch.equal(y[0, 9], b)
    rows[0, 9] = False
    assert torch.equal(y[rows], tk.layer_norm(x, w, b)[rows])
    for shape in ((0, 512), (2, 0, 512)):
        x0, w0 = torch.empty(shape, device=DEV, requires_grad=True), w.clone().requires_grad_(True)
        y0 = tk.layer_norm(x0, w0, b)
        dx0, dw0 = torch.autograd.grad(y0, (x0, w0), torch.empty_like(y0))
        assert y0.shape == dx0.shape == shape and torch.equal(dw0, torch.zeros_like(w))


@pytest.mark.gpu
@pytest.mark.parametrize("n,plus_one", [(384, False), (385, True), (9000, False)])
def test_gradients_against_differences(n, plus_one):
    """(f(+e) - f(-e)) / 2e along a random direction, f = sum(y dy) added up in 64 bits. With e = 2^-6 the step's third-order term is below
    e^2 = 2.5e-4 of the gradient's size times the direction's; the roundings of y, u each over 2e, are 2e-6 of it."""
    (x, dy), g = inputs((2, 21, n), F32, n)
    w, b = randn(g, 2, 1, n).to(DEV), randn(g, n).to(DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(tk.layer_norm(*leaves, plus_one=plus_one), leaves, dy)
    e = 2.0 ** -6
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = randn(g, *leaf.shape).to(DEV)
        v = v / v.norm() * math.sqrt(v.numel())
        with torch.no_grad():
            f = [(tk.layer_norm(*[t + s * e * v if j == i else t for j, t in enumerate(leaves)], plus_one=plus_one).double() * dy.double()).sum() for s in (1, -1)]
        got, want = (grad.double() * v.double()).sum(), (f[0] - f[1]) / (2 * e)
        assert abs(got - want) <= 1e-3 * grad.double().norm() * v.double().norm()


@pytest.mark.gpu
def test_module_and_gradients_into_parameters():
    ours, theirs = tk.LayerNorm(320).to(DEV), torch.nn.LayerNorm(320).to(DEV)
    g = seeded(1)
    with torch.no_grad():
        for p in ours.parameters():
            p.copy_(randn(g, 320))
    theirs.load_state_dict(ours.state_dict())
    x = randn(g, 4, 33, 320).to(DEV)
    for m in (ours, theirs):
        for _ in range(2):
            m(x).square().sum().backward()
    for p, q in zip(ours.parameters(), theirs.parameters()):
        torch.testing.assert_close(p.grad, q.grad, atol=2e-3, rtol=1e-5)     # sums of 132 terms of up to 50: 132 * 50 * 2^-24 * a few
    x = torch.randn(3, 320, device=DEV, requires_grad=True)
    y = tk.layer_norm(x)
    dy = torch.randn(3, 320, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError):      # the gradient is not differentiable itself
        torch.autograd.grad(torch.autograd.grad(y, x, dy, create_graph=True)[0].sum(), dy)
    frozen = tk.layer_norm(x.detach(), torch.ones(320, device=DEV))
    assert not frozen.requires_grad


@pytest.mark.gpu
def test_the_same_bits_again_on_another_stream_and_from_a_graph():
    (x, dy), g = inputs((2, 333, 768), BF, 2)
    w, b = randn(g, 2, 1, 768, dtype=BF).to(DEV), randn(g, 2, 1, 768, dtype=BF).to(DEV)

    def step(x, w, b, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = tk.layer_norm(*leaves, plus_one=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(want, again):
        assert torch.equal(a, c)
    held = [t.clone() for t in (x, w, b, dy)]
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step(*held))
    for i in range(4):
        fresh, _ = inputs((2, 333, 768), BF, 10 + i)
        for t, f in zip((held[0], held[3]), fresh):
            t.copy_(f)
        for graph in graphs:
            graph.replay()
        eager = step(*held)
        for out in outs:
            for a, c in zip(out, eager):
                assert torch.equal(a, c)
        torch.cuda.synchronize()


def test_refusals_need_no_gpu():
    x = torch.zeros(2, 3, 16)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.layer_norm(x)
    with pytest.raises(AssertionError):
        tk.LayerNorm((4, 16))
    m = tk.LayerNorm(16)
    assert set(m.state_dict()) == {"weight", "bias"} and set(tk.LayerNorm(16, bias=False).state_dict()) == {"weight"}
    with pytest.raises(AssertionError):
        m(torch.zeros(2, 8))
    torch.testing.assert_close(tk.layer_norm_torch(x + torch.arange(16.0), m.weight, m.bias), torch.nn.functional.layer_norm(x + torch.arange(16.0), (16,)))


@pytest.mark.gpu
def test_refusals():
    x, w = torch.zeros(2, 3, 16, device=DEV), torch.zeros(16, device=DEV)
    for bad in (torch.zeros(8, device=DEV), torch.zeros(3, 1, 16, device=DEV), torch.zeros(2, 2, 16, device=DEV), torch.zeros((), device=DEV)):
        with pytest.raises(AssertionError):
            tk.layer_norm(x, bad)
        with pytest.raises(AssertionError):
            tk.layer_norm(x, w, bad)
    with pytest.raises(TypeError):
        tk.layer_norm(x.half(), w)
    with pytest.raises(RuntimeError, match="65536"):
        tk.layer_norm(torch.zeros(1, 65537, device=DEV))
    with pytest.raises(RuntimeError, match="different devices|GPU"):
        tk.layer_norm(x, w.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tokens,n", [(2, 63, 96), (1, 128, 3000), (1, 129, 512), (4, 128, 4096), (5, 128, 4096), (64, 8, 320), (70, 3, 1001), (1, 2, 16384), (255, 2, 64), (3, 128, 1003), (300, 1, 72)])
@pytest.mark.parametrize("each", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_few_rows_and_many_weights(batch, tokens, n, each, dtype):
    """Around the bounds of the backward pass in one launch, with any of its outputs left out, and the sums of few parts for many weights."""
    (x, dy), g = inputs((batch, tokens, n), dtype, n + batch)
    w, b = (randn(g, *((batch, 1, n) if each else (n,)), dtype=dtype).to(DEV) for _ in range(2))
    for wanted in ("xwb", "wb", "xw", "b"):
        check(x, w, b, dy, plus_one=each, wanted=wanted)
    check(x, None, b, dy)
