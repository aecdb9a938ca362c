"""Products with weights in 4 bits against the formula in float64, their layout, and what they refuse."""
import math

import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from triton_kernels.kernels import quantization
from util import DEV, randn, seeded

HALF = torch.finfo(torch.bfloat16).eps / 2


def weights(g, n, k, group, zeros, device=DEV):
    q = torch.randint(0, 16, (n, k), generator=g)
    scale = ((0.5 + torch.rand(n, k // group, generator=g)) * 0.3 * k ** -0.5).bfloat16()
    zero = torch.randint(0, 16, (n, k // group), generator=g) if zeros else None
    return tk.pack_w4(q.to(device), scale.to(device), None if zero is None else zero.to(device)), q, scale, zero


def plain_weight(q, scale, zero):
    z = 8.0 if zero is None else zero.double().repeat_interleave(q.shape[1] // scale.shape[1], 1)
    return (q.double() - z) * scale.double().repeat_interleave(q.shape[1] // scale.shape[1], 1)


def gelu(y):
    return y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def expected(x, b, q, scale, zero, activation, in_activation, rounded):
    """The result in float64 and how far a result may be from it, value by value and in the root mean square of all.

    y's rounding is half a step. K + 8 sums and products of fp32 numbers of at most sum |s| (16 + q + 16 + z) |f(x)|, each good to 2^-23 (a product on the matrix
    cores may cut where it does not round). f(x) is held to half a step of half a step, and its exponential and reciprocal are good to 2^-20.
    Weights laid out as bf16 (`rounded`) are half a step off. GELU's slope is at most 1.13, and its own exponential and reciprocal are good to 2^-20."""
    w, xf = plain_weight(q, scale, zero), x.double()
    f = xf * torch.sigmoid(xf) if in_activation else xf
    y = f @ w.T + (0 if b is None else b.double())
    group = q.shape[1] // scale.shape[1]
    reach = (32.0 + q.double() + (8.0 if zero is None else zero.double().repeat_interleave(group, 1))) * scale.double().repeat_interleave(group, 1)
    size = f.abs() @ reach.T + (0 if b is None else b.double().abs())
    terms, power = f.abs() @ w.abs().T, (f ** 2 @ (w ** 2).T).sqrt()
    slope = 1.13 if activation else 1.0
    off = slope * ((q.shape[1] + 8) * 2.0 ** -23 * size + (terms * (HALF ** 2 + 2.0 ** -19) if in_activation else 0) + (terms * HALF if rounded else 0))
    # the same in the mean: independent errors add by their squares, a rounding is spread evenly over its half step
    mean = slope * (q.shape[1] ** 0.5 * 2.0 ** -23 * size + (terms * (HALF ** 2 + 2.0 ** -19) if in_activation else 0) + (power * HALF / 3 ** 0.5 if rounded else 0))
    if activation:
        y, off, mean = gelu(y), off + 2.0 ** -19 * y.abs(), mean + 2.0 ** -19 * y.abs()
    return y, off + HALF * (y.abs() + off), ((HALF / 3 ** 0.5 * y.abs()) ** 2 + mean ** 2).mean().sqrt() * 1.25


def check(got, x, b, q, scale, zero, activation="", in_activation="", rounded=False):
    want, off, mean = expected(x.cpu(), None if b is None else b.cpu(), q, scale, zero, activation, in_activation, rounded)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= off).all()), f"{(err - off).max().item():.3e} beyond the bound"
    if want.numel() >= 256:
        assert err.pow(2).mean().sqrt() <= mean


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,rows,n,k", [(32, 1, 1, 32), (64, 1, 17, 64), (128, 1, 16, 128), (32, 2, 100, 160), (64, 3, 257, 448), (128, 5, 48, 3072), (64, 8, 33, 8256), (32, 9, 130, 96), (128, 15, 31, 640),
                                            (64, 16, 96, 2048), (32, 17, 64, 4096), (64, 33, 40, 192), (128, 63, 144, 384), (64, 64, 20, 3072), (64, 65, 80, 320), (32, 32, 48, 8224), (64, 40, 100, 8256), (128, 128, 2100, 1152), (64, 12, 4200, 1088), (64, 24, 9000, 64), (32, 4, 300, 8192), (64, 100, 9300, 128), (128, 129, 64, 256), (32, 130, 264, 1056), (128, 257, 128, 1024)])
def test_against_float64(group, rows, n, k, zeros):
    g = seeded(rows * n + k)
    w, q, scale, zero = weights(g, n, k, group, zeros)
    x, b = randn(g, rows, k, dtype=torch.bfloat16), randn(g, n, dtype=torch.bfloat16)
    check(tk.linear_w4(x.to(DEV), w, b.to(DEV)), x, b, q, scale, zero, rounded=rows > 128)
    check(tk.linear_w4(x.to(DEV), w, activation="GELU"), x, None, q, scale, zero, "GELU", rounded=rows > 128)


@pytest.mark.gpu
@pytest.mark.parametrize("group,rows,n,k,zeros", [(64, 1, 512, 3072, False), (128, 3, 100, 1024, True), (32, 8, 65, 2080, True), (64, 8, 16, 8256, False), (32, 5, 1, 32, False), (64, 2, 48, 64, True), (64, 5, 4200, 320, True), (32, 3, 5000, 96, False), (128, 4, 100, 8192, True)])
def test_silu_on_the_way_in(group, rows, n, k, zeros):
    g = seeded(rows + n + k)
    w, q, scale, zero = weights(g, n, k, group, zeros)
    x, b = randn(g, rows, k, dtype=torch.bfloat16, std=2.0), randn(g, n, dtype=torch.bfloat16)
    check(tk.linear_w4(x.to(DEV), w, b.to(DEV), in_activation="SiLU"), x, b, q, scale, zero, "", "SiLU")
    check(tk.linear_w4(x.to(DEV), w, b.to(DEV), in_activation="SiLU", activation="GELU"), x, b, q, scale, zero, "GELU", "SiLU")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 20, 70, 140])
@pytest.mark.parametrize("silu", [False, True])
def test_what_is_not_finite_goes_as_in_the_formula(rows, silu):
    if silu and rows > 8:
        pytest.skip("the input activation is for at most 8 rows")
    g = seeded(rows)
    w, q, scale, zero = weights(g, 40, 256, 64, True)
    x = randn(g, rows, 256, dtype=torch.bfloat16)
    x[0, 3], x[rows - 1, 200] = math.inf, 1e36   # (15 times which is still a number in fp32)
    if rows > 8:
        x[5, 17], x[6, 100], x[7, 0] = -math.inf, math.nan, -1e36
    got = tk.linear_w4(x.to(DEV), w, in_activation="SiLU" if silu else "").double().cpu()
    want = expected(x, None, q, scale, zero, "", "SiLU" if silu else "", False)[0]
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf() & (got > 0), want.isinf() & (want > 0)) and torch.equal(got.isinf() & (got < 0), want.isinf() & (want < 0))
    fine = want.isfinite()
    assert bool(want.isinf().any()) and bool(want.isnan().any()) and (rows == 1 or bool(fine.any()))
    assert torch.allclose(got[fine], want[fine], rtol=3 * HALF, atol=0.05)   # beside the exact check of finite rows above


@pytest.mark.gpu
def test_views_and_leading_dimensions():
    g = seeded(5)
    w, q, scale, zero = weights(g, 48, 192, 64, False)
    wide = randn(g, 2, 5, 3 * 192 + 8, dtype=torch.bfloat16).to(DEV)
    for x in (wide[..., 192:384], wide[..., 3:195], wide[:, :3, 8:200], wide[:, ::2, :192], wide[..., :384:2], wide[0, 0, :192], wide[1, :, 8:200], wide[:, 0, None, 16:208]):
        y = tk.linear_w4(x, w)
        assert y.shape == (*x.shape[:-1], 48) and y.is_contiguous()
        check(y.reshape(-1, 48), x.reshape(-1, 192), None, q, scale, zero)
    assert tk.linear_w4(wide[:0, :, :192], w).shape == (0, 5, 48)
    b = randn(g, 96, dtype=torch.float32).to(DEV)[::2]   # another type and stride of the bias
    check(tk.linear_w4(wide[0, :, :192], w, b), wide[0, :, :192], b.bfloat16(), q, scale, zero)


@pytest.mark.gpu
@pytest.mark.parametrize("group,n,k,zeros", [(32, 1, 32, True), (64, 33, 448, False), (128, 100, 1152, True)])
def test_the_weight_itself(group, n, k, zeros):
    w, q, scale, zero = weights(seeded(n), n, k, group, zeros)
    assert torch.equal(w.dequantize().cpu(), plain_weight(q, scale, zero).bfloat16())


@pytest.mark.gpu
def test_rows_are_the_same_whoever_stands_beside_them():
    g = seeded(11)
    w, *_ = weights(g, 64, 512, 64, True)
    x = randn(g, 16, 512, dtype=torch.bfloat16).to(DEV)
    alone, together = tk.linear_w4(x[3:4], w), tk.linear_w4(x, w)
    assert torch.equal(alone[0], together[3])
    x[4] = math.nan
    assert torch.equal(tk.linear_w4(x[:4], w), together[:4])


@pytest.mark.gpu
def test_streams_and_replayed_graphs():
    g = seeded(12)
    w, q, scale, zero = weights(g, 96, 256, 64, False)
    x = randn(g, 140, 256, dtype=torch.bfloat16).to(DEV)
    want = [tk.linear_w4(x[:r], w) for r in (1, 40, 140)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = [tk.linear_w4(x[:r], w) for r in (1, 40, 140)]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph, again = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = [tk.linear_w4(again[:r], w) for r in (1, 40, 140)]
    for i in range(3):
        again.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, tk.linear_w4((x * (i + 1))[:r], w)) for a, r in zip(out, (1, 40, 140)))


@pytest.mark.gpu
def test_gradients_are_an_error():
    w, *_ = weights(seeded(1), 32, 64, 32, False)
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError):
        tk.linear_w4(x, w).sum().backward()
    b = torch.zeros(32, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError):
        tk.linear_w4(x.detach(), w, b).sum().backward()
    with torch.no_grad():
        assert not tk.linear_w4(x, w, b).requires_grad


@pytest.mark.gpu
def test_refusals_of_a_call():
    w, *_ = weights(seeded(1), 32, 64, 32, False)
    x = torch.zeros(9, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(AssertionError):
        tk.linear_w4(x[:, :32], w)
    with pytest.raises(TypeError):
        tk.linear_w4(x.float(), w)
    with pytest.raises(KeyError):
        tk.linear_w4(x, w, activation="ReLU")
    with pytest.raises(KeyError):
        tk.linear_w4(x, w, in_activation="GELU")
    with pytest.raises(NotImplementedError):
        tk.linear_w4(x, w, in_activation="SiLU")
    with pytest.raises(AssertionError):
        tk.linear_w4(x, w, torch.zeros(31, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError):
        tk.linear_w4(x, w.to("cpu"))
    with pytest.raises(RuntimeError):
        tk.linear_w4(x.cpu(), w)


def test_layout_is_the_headers():
    g = seeded(3)
    for n, k, group, zeros in [(1, 32, 32, False), (17, 96, 32, True), (40, 192, 64, True), (33, 384, 128, True)]:
        w, q, scale, zero = weights(g, n, k, group, zeros, "cpu")
        assert w.shape == (n, k) and w.packed.shape == (-(-n // 16), -(-k // 128), 1024)
        for i, j in [(0, 0), (n - 1, k - 1)] + [(int(a * n), int(b * k)) for a, b in torch.rand(40, 2, generator=g).tolist()]:
            at, c, e = j % 128 // 32, j % 32 // 8, j % 8
            word = int.from_bytes(bytes(w.packed[i // 16, j // 128].view(4, 16, 16)[c, i % 16, 4 * at:4 * at + 4].tolist()), "little")
            assert word >> 4 * (e // 2) + 16 * (e % 2) & 15 == q[i, j]
            assert w.scale[i // 16, j // 128, i % 16, j % 128 // group] == scale[i, j // group]
            assert zero is None or w.zero[i // 16, j // 128, i % 16, j % 128 // group] == zero[i, j // group]
        back = w.unpack()
        assert torch.equal(back[0].long(), q) and torch.equal(back[1], scale) and (zero is None or torch.equal(back[2].long(), zero))


def test_quantised_weights_are_the_nearest():
    g = seeded(4)
    wf = randn(g, 24, 256)
    wf[3, 64:128], wf[4] = 0.0, wf[4].abs()
    for zeros in (False, True):
        w = tk.quantize_w4(wf, 64, zeros)
        q, scale, zero = w.unpack()
        got, step = plain_weight(q, scale, zero), scale.double().repeat_interleave(64, 1)
        assert bool((got[3, 64:128] == 0).all())
        # half a step; at an end the scale's own rounding (half of a bf16 step of 15 or 8 of them) and, with zero points, that of the zero
        ends = 8 * HALF if not zeros else 15 * HALF + 0.5
        assert bool(((got - wf.double()).abs() <= step * (0.5 + ends)).all())
    whole = (torch.randint(0, 16, (8, 64), generator=g).float() - 8) * 0.25
    whole[:, 0] = -8 * 0.25 * 7.5 / 8
    q = tk.quantize_w4(whole, 32).unpack()[0]
    assert int(q.min()) >= 0 and int(q.max()) <= 15


def test_refusals_of_a_layout():
    q, s = torch.zeros(4, 64, dtype=torch.int64), torch.zeros(4, 1, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        tk.pack_w4(q + 16, s)
    with pytest.raises(ValueError):
        tk.pack_w4(q - 1, s)
    with pytest.raises(TypeError):
        tk.pack_w4(q.float(), s)
    with pytest.raises(TypeError):
        tk.pack_w4(q, s.float())
    with pytest.raises(AssertionError):
        tk.pack_w4(q[:, :48], s)
    with pytest.raises(AssertionError):
        tk.pack_w4(q, s[:3])
    with pytest.raises(AssertionError):
        tk.pack_w4(q, s, torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(ValueError):
        tk.pack_w4(q, s, torch.full((4, 1), 16))
    with pytest.raises(AssertionError):
        tk.quantize_w4(torch.zeros(4, 48))
    with pytest.raises(ValueError):
        tk.quantize_w4(torch.full((4, 64), math.nan))
    w = tk.pack_w4(q, s)
    with pytest.raises(AssertionError):
        quantization.W4(w.packed, w.scale, w.zero, (20, 64), 64)
    with pytest.raises(AssertionError):
        quantization.W4(w.packed.long(), w.scale, w.zero, (4, 64), 64)
    with pytest.raises(RuntimeError):
        w.dequantize()


@pytest.mark.parametrize("change,rc", [(dict(x=None), -1), (dict(y=None), -1), (dict(M=-1), -2), (dict(act=2), -6), (dict(in_act=1), -6), (dict(in_act=2, M=9), -6), (dict(M=0, x=None), 0), (dict(x=24), -4),
                                       (dict(M=2, ldx=65), -4), (dict(M=2, ldy=3), -2), (dict(M=129), -2)])
def test_refusals_of_the_library(change, rc):
    import ctypes

    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    w = nv.W4(p, p, None, 16, 64, 64)
    a = nv.LinearW4Args(**{**dict(x=p, bias=None, y=p, w=w, M=1, ldx=64, ldy=16, act=0, in_act=0), **change})
    if a.x is not None and a.x < 4096:
        a.x = p + 8
    assert nv.lib().flux_linear_w4_bf16(ctypes.byref(a), None, 0, None) == rc
    assert nv.lib().flux_linear_w4_bf16(None, None, 0, None) == -1
    for bad, code in ((nv.W4(p, p, None, 16, 64, 48), -6), (nv.W4(p, p, None, 16, 96, 64), -2), (nv.W4(p, p, None, -1, 64, 64), -2), (nv.W4(None, p, None, 16, 64, 64), -1), (nv.W4(p + 8, p, None, 16, 64, 64), -4)):
        b = nv.LinearW4Args(p, None, p, bad, 1, 64, 16, 0, 0)
        assert nv.lib().flux_linear_w4_bf16(ctypes.byref(b), None, 0, None) == code
        assert nv.lib().flux_w4_unpack(ctypes.byref(bad), p, None) == code


# Beyond 128 rows, thousands of outputs: weights unpacked between the products. Fewer columns than a slab of 128, ends of slabs, more than the ring of four holds; last workgroups of one row
# and of a few outputs, two and three tiles a wave.
@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,rows,n,k", [(32, 129, 9301, 96), (64, 256, 9216, 192), (128, 200, 12300, 640), (64, 385, 6200, 1088), (32, 512, 9217, 32), (64, 513, 7000, 320), (128, 640, 9000, 1152), (32, 1000, 4616, 160)])
def test_hundreds_of_rows_of_thousands_of_outputs(group, rows, n, k, zeros):
    g = seeded(rows + n + k)
    w, q, scale, zero = weights(g, n, k, group, zeros)
    wide = randn(g, rows, k + 24, dtype=torch.bfloat16)
    wide[:, k:], wide[:, :8] = math.nan, math.inf   # (what lies beside a row is not its own)
    x, b = wide[:, 8:k + 8].clone(), randn(g, n, dtype=torch.bfloat16)
    wide[:, 8:k + 8] = x[:] = randn(g, rows, k, dtype=torch.bfloat16)
    moved = wide.to(DEV)
    check(tk.linear_w4(moved[:, 8:k + 8], w, b.to(DEV)), x, b, q, scale, zero, rounded=True)
    check(tk.linear_w4(x.to(DEV), w, activation="GELU"), x, None, q, scale, zero, "GELU", rounded=True)


@pytest.mark.gpu
def test_hundreds_of_rows_that_are_not_finite():
    g = seeded(31)
    w, q, scale, zero = weights(g, 9216, 256, 64, True)
    x = randn(g, 200, 256, dtype=torch.bfloat16)
    x[0, 3], x[199, 255], x[130, 17], x[131, 100] = math.inf, -math.inf, math.nan, 1e36
    got = tk.linear_w4(x.to(DEV), w).double().cpu()
    want = expected(x, None, q, scale, zero, "", "", True)[0]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf() & (got > 0), want.isinf() & (want > 0)) and torch.equal(got.isinf() & (got < 0), want.isinf() & (want < 0))
    rest = [i for i in range(200) if i not in (0, 130, 131, 199)]
    # scales from the smallest to nearly the largest, whose products with q - z are numbers
    for size in (2.0 ** -133, 2.0 ** -126, 2.0 ** 123):
        most = tk.pack_w4(q, torch.full_like(scale, size), zero).to(DEV)
        assert torch.equal(tk.linear_w4(torch.eye(256, dtype=torch.bfloat16, device=DEV), most).t(), most.dequantize())
    check(tk.linear_w4(x.to(DEV), w)[rest], x[rest], None, q, scale, zero, rounded=True)


@pytest.mark.gpu
def test_hundreds_of_rows_in_a_graph_and_on_a_stream():
    g = seeded(32)
    w, *_ = weights(g, 9216, 384, 64, False)
    x = randn(g, 300, 384, dtype=torch.bfloat16).to(DEV)
    stream = torch.cuda.Stream()
    want = [tk.linear_w4(x * i, w) for i in (1, 2, 3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        other = tk.linear_w4(x, w)
    stream.synchronize()
    assert torch.equal(other, want[0])
    graph, mine = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = tk.linear_w4(mine, w)
    for i in range(3):
        mine.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
