"""apply_rope_nd and rope_table against the formulas in 64 bits.

Tolerances. Sines and cosines are off by at most 2^-23: 2^-25 |x| for the reduced angle's rounding, two roundings of the series and its rest. An angle
in 64 bits carries the roundings of the frequency (up to d / 16 + 2 multiplications) and of the product, 2^-53 each. A turned value is the sum
of two products, each rounded, and is rounded to its type once more."""
import pytest
import torch

import triton_kernels as tk
from triton_kernels import flux
from triton_kernels import testing as cfg
from util import DEV, randn, seeded

BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def angles(ids, axes, theta):
    """[B or 1, 1, L, pairs] in 64 bits, and how far each may be off."""
    ids = ids.double() if ids.dim() == 3 else ids.double()[None]
    out = [ids[..., i] / theta ** (2.0 * j / d) for i, d in enumerate(axes) for j in range(d // 2)]
    angle = torch.stack(out, -1).unsqueeze(1)
    return angle, angle.abs() * (max(axes) / 16 + 4) * 2.0 ** -52 + 2.0 ** -23


def turned(x, angle, off):
    x = x.double().unflatten(-1, (-1, 2))
    c, s = angle.cos(), angle.sin()
    want = torch.stack((x[..., 0] * c - x[..., 1] * s, x[..., 0] * s + x[..., 1] * c), -1).flatten(-2)
    size = x.abs().sum(-1)
    return want, (size * (off + 2.0 ** -23)).repeat_interleave(2, -1)


def near(got, x, angle, off):
    want, bound = turned(x, angle, off)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert ((got.double() - want).abs() <= bound + HALF_STEP[x.dtype] * want.abs()).all(), (got.double() - want).abs().max()


def check(q, k, ids, axes, theta=10000.0):
    angle, off = angles(ids, axes, theta)
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    outs = tk.apply_rope_nd(*leaves, ids, axes, theta)
    for x, y in zip((q, k), outs):
        near(y, x, angle, off)
    dys = [torch.flip(x, (0, 3)).contiguous() for x in (q, k)]
    for dy, dx in zip(dys, torch.autograd.grad(outs, leaves, dys)):
        near(dx, dy, -angle, off)
    table = tk.rope_table(ids, axes, theta)
    assert table.shape == (*angle.shape, 2, 2) and table.dtype == F32
    assert ((table[..., 0, 0].double() - angle.cos()).abs() <= off).all() and ((table[..., 1, 0].double() - angle.sin()).abs() <= off).all()
    assert torch.equal(table[..., 0, 0], table[..., 1, 1]) and torch.equal(table[..., 0, 1], -table[..., 1, 0])


def video(B, frames, height, width, text=0, axes=3):
    grid = torch.cartesian_prod(torch.arange(frames), torch.arange(height), torch.arange(width)).double().reshape(-1, 3)[:, 3 - axes:]
    ids = torch.cat((torch.zeros(text, axes).double(), grid))
    return torch.stack([ids + 5 * b for b in range(B)]).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("axes", [(16, 56, 56), (32, 48, 48), (64,), (44, 42, 42), (24, 12, 12), (2, 2), (6,), (8, 8, 8, 8, 8, 8, 8, 8), (64, 96, 96), (128, 192, 192), (10, 250), (2, 508, 2)])
@pytest.mark.parametrize("B,heads,kv,L", [(1, 24, 24, 37), (3, 5, 1, 1), (2, 1, 9, 130)])
def test_shapes(B, heads, kv, L, axes, dtype):
    g = seeded(B + heads + L + sum(axes))
    ids = torch.randint(-40, 300, (B, L, len(axes)), generator=g).double().to(DEV)
    q, k = randn(g, B, heads, L, sum(axes), dtype=dtype).to(DEV), randn(g, B, kv, L, sum(axes), dtype=dtype).to(DEV)
    check(q, k, ids, axes)


@pytest.mark.gpu
@pytest.mark.parametrize("ids_dtype", [F32, torch.float64, torch.int32, torch.int64, BF, torch.int16])
def test_types_and_shapes_of_ids(ids_dtype):
    g = seeded(2)
    q, k = randn(g, 2, 3, 60, 64).to(DEV), randn(g, 2, 2, 60, 64).to(DEV)
    ids = video(2, 3, 4, 5).to(ids_dtype)
    for at in (ids, ids[:1], ids[0], ids.repeat_interleave(2, 2)[..., ::2], ids.transpose(0, 1).contiguous().transpose(0, 1), ids.flip(1)):
        check(q, k, at, (16, 24, 24), 256)
    if ids_dtype.is_floating_point:
        check(q, k, ids / 4 + 0.5, (16, 24, 24))


@pytest.mark.gpu
@pytest.mark.parametrize("far", [1e4, 1e6, 2.0 ** 30])
def test_far_positions(far):
    """Angles of millions of radians keep the accuracy of a near one: 2^30 * (8 + 4) * 2^-52 = 3e-6 at worst."""
    g = seeded(4)
    q, k = randn(g, 1, 2, 64, 128).to(DEV), randn(g, 1, 2, 64, 128).to(DEV)
    ids = (far + 77 * torch.arange(64 * 3).double()).round().view(1, 64, 3).to(DEV)
    check(q, k, ids, (16, 56, 56))
    check(q, k, -ids, (16, 56, 56))
    check(q, k, ids.long(), (64, 32, 32), 1e6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_alignment(dtype):
    """Views of a fused projection, of a text and an image part, with a strided last dimension, at odd addresses, broadcast."""
    g = seeded(6)
    ids = video(2, 2, 4, 5, text=3)
    fused = randn(g, 2, 50, 14, 72, dtype=dtype).to(DEV)
    heads = fused.transpose(1, 2)
    axes = (24, 24, 24)
    check(heads[:, :8, :43], heads[:, 8:10, :43], ids, axes)
    check(heads[:, 3:4, 7:], heads[:, 4:14:3, 7:], ids, axes)
    check(heads[:, :4, :43].transpose(2, 3).contiguous().transpose(2, 3), heads[:, :4, :43], ids, axes)
    odd = fused.reshape(2, 50, 14 * 72)[:, :43, 1:1 + 3 * 66].unflatten(-1, (3, 66)).transpose(1, 2)
    check(odd, odd[:, :1], ids, (22, 22, 22))
    check(heads[:, :1, :43].expand(2, 6, 43, 72), heads[:1, :2, :43].expand(2, 2, 43, 72), ids, axes)


@pytest.mark.gpu
def test_what_apply_rope_and_embed_nd_do():
    """Beside the plain blocks' EmbedND and apply_rope with its table: two roundings of the table's entries apart."""
    g = seeded(8)
    ids = cfg.flux_position_ids(32, 16).to(DEV)
    q, k = randn(g, 1, 4, 288, 128).to(DEV), randn(g, 1, 4, 288, 128).to(DEV)
    plain, ours = flux.EmbedND(128, 10000, [16, 56, 56])(ids), tk.EmbedND(128, 10000, [16, 56, 56])(ids)
    assert ours.shape == plain.shape
    torch.testing.assert_close(ours, plain, atol=2.0 ** -23 + 2.0 ** -25, rtol=0)
    for got, want in zip(tk.apply_rope_nd(q, k, ids, [16, 56, 56]), tk.apply_rope(q, k, ours)):
        torch.testing.assert_close(got, want, atol=2.0 ** -22 * 10, rtol=0)     # |x0| + |x1| < 10
    assert torch.equal(tk.rope_table(ids[0], (16, 56, 56)), ours)


@pytest.mark.gpu
def test_without_k_without_rows_and_not_finite():
    g = seeded(9)
    ids = video(1, 1, 3, 4)
    q = randn(g, 1, 3, 12, 64).to(DEV).requires_grad_(True)
    yq, yk = tk.apply_rope_nd(q, None, ids, (16, 24, 24))
    assert yk is None and torch.equal(yq, tk.apply_rope_nd(q, q, ids, (16, 24, 24))[1])
    k = q.detach().clone().requires_grad_(True)
    out = tk.apply_rope_nd(q, k, ids, (16, 24, 24))
    dk, = torch.autograd.grad(out[1].sum(), k)                      # one of the two outputs alone, one input alone
    dq, = torch.autograd.grad(tk.apply_rope_nd(q, k.detach(), ids, (16, 24, 24))[0].sum(), q)
    assert torch.equal(dq, dk)
    bad = q.detach().clone()
    bad[0, 1, 5, 9], bad[0, 2, 7, 20] = float("nan"), float("inf")
    y = tk.apply_rope_nd(bad, None, ids, (16, 24, 24))[0]
    want = torch.ones_like(y, dtype=torch.bool)
    want[0, 1, 5, 8:10] = want[0, 2, 7, 20:22] = False
    assert torch.equal(y.isfinite(), want) and torch.equal(y[want], yq.detach()[want])
    for B, L in ((0, 4), (2, 0)):
        empty = torch.empty(B, 3, L, 64, device=DEV, requires_grad=True)
        at = torch.zeros(B, L, 3, device=DEV)
        a, b = tk.apply_rope_nd(empty, empty, at, (16, 24, 24))
        assert a.shape == b.shape == empty.shape and torch.autograd.grad(a.sum(), empty)[0].shape == empty.shape
        assert tk.rope_table(at, (16, 24, 24)).shape == (B, 1, L, 32, 2, 2)


@pytest.mark.gpu
def test_gradients_against_differences():
    """The operator is linear in x: (f(x + v) - f(x - v)) / 2 = f'(x) v up to the roundings of f, 2^-23 of the values' sizes summed over 2 x 2880 of them."""
    g = seeded(12)
    ids = video(1, 1, 3, 5, text=0)
    x, v, dy = (randn(g, 1, 3, 15, 64).to(DEV) for _ in range(3))
    leaf = x.clone().requires_grad_(True)
    grad, = torch.autograd.grad(tk.apply_rope_nd(leaf, None, ids, (16, 24, 24))[0], leaf, dy, create_graph=True)
    f = [(tk.apply_rope_nd(x + s * v, None, ids, (16, 24, 24))[0].double() * dy.double()).sum() for s in (1, -1)]
    assert abs((f[0] - f[1]) / 2 - (grad.double() * v.double()).sum()) <= 2880 * 2 * 2.0 ** -23 * 10
    twice = dy.clone().requires_grad_(True)                          # and it can be differentiated again
    grad, = torch.autograd.grad(tk.apply_rope_nd(leaf, None, ids, (16, 24, 24))[0], leaf, twice, create_graph=True)
    back, = torch.autograd.grad(grad, twice, v)
    assert torch.equal(back, tk.apply_rope_nd(v, None, ids, (16, 24, 24))[0])


@pytest.mark.gpu
def test_another_stream_and_graphs():
    g = seeded(13)
    ids = video(2, 2, 5, 7, text=4)
    q, k = randn(g, 2, 74, 3, 64, dtype=BF).to(DEV).transpose(1, 2), randn(g, 2, 74, 3, 64, dtype=BF).to(DEV).transpose(1, 2)
    want = tk.apply_rope_nd(q, k, ids, (16, 24, 24))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = tk.apply_rope_nd(q, k, ids, (16, 24, 24))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (*tk.apply_rope_nd(q, k, ids, (16, 24, 24)), tk.rope_table(ids, (16, 24, 24)))
    for i in range(3):
        ids.add_(3)
        q.copy_(randn(g, *q.shape, dtype=BF))
        graph.replay()
        eager = (*tk.apply_rope_nd(q, k, ids, (16, 24, 24)), tk.rope_table(ids, (16, 24, 24)))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        torch.cuda.synchronize()


def test_refusals_need_no_gpu():
    q, ids = torch.zeros(1, 2, 4, 64), torch.zeros(1, 4, 3)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.apply_rope_nd(q, q, ids, (16, 24, 24))
    with pytest.raises(RuntimeError, match="GPU"):
        tk.rope_table(ids, (16, 24, 24))
    for bad in ((q, q, ids, (16, 24, 26)), (q[0], q[0], ids, (16, 24, 24)), (q, q.double(), ids, (16, 24, 24)), (q, q[:, :, :3], ids, (16, 24, 24)), (q, q[..., :32], ids, (16, 24, 24))):
        with pytest.raises(AssertionError):
            tk.apply_rope_nd(*bad)
    a, b = tk.apply_rope_nd_torch(q + 1, q[:, :1] + 1, ids, (16, 24, 24))
    assert a.shape == q.shape and b.shape == (1, 1, 4, 64) and torch.equal(a, q + 1)


@pytest.mark.gpu
def test_refusals():
    q, ids = torch.zeros(2, 2, 4, 64, device=DEV), torch.zeros(2, 4, 3, device=DEV)
    for bad in (ids[..., :2], ids[:, :3], torch.zeros(3, 4, 3, device=DEV), ids[None], ids[0, 0]):
        with pytest.raises(AssertionError):
            tk.apply_rope_nd(q, q, bad, (16, 24, 24))
    with pytest.raises(AssertionError):
        tk.apply_rope_nd(q, q, ids, (15, 24, 25))
    with pytest.raises(AssertionError):
        tk.rope_table(ids, (16, 24))
    with pytest.raises(TypeError):
        tk.apply_rope_nd(q.half(), q.half(), ids, (16, 24, 24))
    with pytest.raises(TypeError):
        tk.apply_rope_nd(q, q, ids.bool(), (16, 24, 24))
    with pytest.raises(ValueError, match="theta"):
        tk.apply_rope_nd(q, q, ids, (16, 24, 24), theta=0.0)
    with pytest.raises(ValueError, match="512"):
        tk.rope_table(ids, (512, 2, 2))
    with pytest.raises(NotImplementedError, match="positions"):
        tk.apply_rope_nd(q, q, ids.clone().requires_grad_(True), (16, 24, 24))
    with pytest.raises(RuntimeError, match="different devices|GPU"):
        tk.apply_rope_nd(q, q, ids.cpu(), (16, 24, 24))
