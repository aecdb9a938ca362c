"""linear_lora against the formula in 64 bits.

Tolerances. u = 2^-24. A sum of K products in fp32 is off by at most K u of the sum of their magnitudes, wherever it is cut. s x a^T is rounded to bf16,
2^-8 of its value, before it meets b; the result once more. GELU's slope is at most 1.13, its own evaluation is good to 2^-18 of |y| + 2^-30."""
import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded

BF, U = torch.bfloat16, 2.0 ** -24


def exact(x, w, b, lora_a, lora_b, adapter, scaling, gelu):
    """The result in 64 bits and how far it may be off."""
    K = x.shape[-1]
    rows = x.reshape(-1, K).double()
    y, off = rows @ w.double().T, K * U * (rows.abs() @ w.double().abs().T)
    if b is not None:
        y, off = y + b.double(), off + 2 * U * b.double().abs()
    owner = adapter.reshape(-1).repeat_interleave(rows.shape[0] // max(1, adapter.numel()))
    for i in range(lora_a.shape[0]):
        at = (owner == i).nonzero()[:, 0]
        s = 1.0 if scaling is None else float(scaling[i])
        a, bt = lora_a[i].double().T, lora_b[i].double().T
        low = s * (rows[at] @ a)
        low_off = 2.0 ** -8 * low.abs() + 2 * K * U * abs(s) * (rows[at].abs() @ a.abs())
        y[at] += low @ bt
        off[at] += low_off @ bt.abs() + lora_a.shape[1] * U * (low.abs() @ bt.abs())
    off = off + 4 * U * y.abs()
    if gelu:
        y, off = torch.nn.functional.gelu(y, approximate="tanh"), 1.13 * off + 2.0 ** -18 * y.abs() + 2.0 ** -30
    return y.view(*x.shape[:-1], -1), off.view(*x.shape[:-1], -1)


def make(seed, lead, K, N, adapters, rank):
    g = seeded(seed)
    x, w, b = randn(g, *lead, K, dtype=BF).to(DEV), randn(g, N, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, N, dtype=BF).to(DEV)
    lora_a, lora_b = randn(g, adapters, rank, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, adapters, N, rank, dtype=BF, std=rank ** -0.5).to(DEV)
    return g, x, w, b, lora_a, lora_b, (0.5 + torch.rand(adapters, generator=g)).to(DEV)


def check(x, w, b, lora_a, lora_b, adapter, scaling, act=""):
    got = tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling, activation=act)
    want, off = exact(x, w, b, lora_a, lora_b, adapter, scaling, act == "GELU")
    assert got.shape == want.shape and got.dtype == BF and not got.requires_grad
    err = (got.double() - want).abs()
    assert (err <= off + 2.0 ** -8 * want.abs()).all(), (err - off - 2.0 ** -8 * want.abs()).max()
    return got


# rows vectors, eight-wave tiles with K whole and in parts, large tiles, whole rounds of them with rows left over, no 16-byte rows
SHAPES = [(1, 64, 40), (3, 1024, 640), (8, 200, 4096), (5, 4096, 96), (7, 8192, 1000), (9, 64, 64), (33, 512, 512), (64, 4096, 1024), (64, 16384, 2048), (150, 1000, 777),
          (517, 2048, 2048), (1100, 256, 1536), (2304, 1024, 3001), (4096, 512, 4096), (6000, 200, 3001), (12, 63, 50), (3, 130, 17), (70, 1001, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_an_adapter_by_row(M, K, N):
    g, x, w, b, lora_a, lora_b, scaling = make(M + K + N, (M,), K, N, 5, 16)
    runs = torch.randint(-2, 7, (M,), generator=g).sort().values.to(DEV)           # runs of rows; -2, -1, 5 and 6 are none
    mixed = torch.randint(-1, 5, (M,), generator=g, dtype=torch.int32).to(DEV)
    check(x, w, b, lora_a, lora_b, runs, scaling)
    check(x, w, None, lora_a, lora_b, mixed, None, "GELU")


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 3, 4, 8, 12, 16, 31, 32, 33, 64, 72, 100, 128, 250, 256])
@pytest.mark.parametrize("B,L,K,N", [(3, 1, 512, 384), (4, 10, 768, 520), (3, 700, 512, 1024)])
def test_ranks(B, L, K, N, rank):
    g, x, w, b, lora_a, lora_b, scaling = make(rank + L, (B, L), K, N, 3, rank)
    check(x, w, b, lora_a, lora_b, torch.tensor([2, 0, -1, 1][:B], device=DEV), scaling, "GELU")
    check(x, w, b, lora_a, lora_b, torch.tensor([1, 1, 1, 1][:B], device=DEV), scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 5, 7, 15, 16, 17, 47, 250, 1111])
def test_requests_of_any_length(L):
    """Requests that begin anywhere in a tile; numbers for the batch, for every row, and one for all."""
    g, x, w, b, lora_a, lora_b, scaling = make(L, (9, L), 384, 800, 6, 24)
    per_request = torch.tensor([5, 0, 0, -1, 3, 3, 1, 9, 5], device=DEV)
    a = check(x, w, b, lora_a, lora_b, per_request, scaling)
    by_row = check(x, w, b, lora_a, lora_b, per_request[:, None].expand(9, L), scaling)
    assert torch.equal(a, by_row)
    check(x, w, b, lora_a, lora_b, torch.tensor(4, device=DEV), scaling)
    check(x, w, b, lora_a, lora_b, per_request.to(torch.int8), scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [20, 200, 1024])
def test_more_adapters_than_rows_in_a_tile(M):
    g, x, w, b, lora_a, lora_b, scaling = make(M, (M,), 256, 320, 300, 8)
    check(x, w, b, lora_a, lora_b, torch.randperm(max(M, 300), generator=g)[:M].to(DEV) % 300, scaling)
    check(x, w, b, lora_a, lora_b, torch.arange(M, device=DEV).flip(0) % 300, scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(64, 512, 1000), (517, 2048, 2048), (64, 16384, 2048), (2500, 512, 4096), (6000, 200, 3001)])
def test_without_adapters_it_is_linear(M, K, N):
    g, x, w, b, lora_a, lora_b, scaling = make(M, (M,), K, N, 2, 16)
    for act in ("", "GELU"):
        assert torch.equal(tk.linear_lora(x, w, b, lora_a, lora_b, torch.full((M,), -1, device=DEV), scaling, act), tk.linear(x, w, b, act))
        zero = tk.linear_lora(x, w, b, lora_a, torch.zeros_like(lora_b), torch.zeros(M, dtype=torch.int32, device=DEV), scaling, act)
        assert torch.equal(zero, tk.linear(x, w, b, act))


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [5, 16, 40])
@pytest.mark.parametrize("M,K,N", [(6, 512, 520), (40, 512, 520), (64, 16384, 2048), (700, 512, 1536), (2500, 256, 4096), (30, 100, 33)])
def test_what_is_not_finite_stays_with_its_rows(M, K, N, rank):
    g, x, w, b, lora_a, lora_b, scaling = make(M + rank, (M,), K, N, 4, rank)
    adapter = torch.randint(-1, 4, (M,), generator=g).to(DEV)
    adapter[0], adapter[1] = 1, 2
    clean = tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling)
    nan, inf = float("nan"), float("inf")
    mine = adapter == 1
    for value in (nan, inf, -inf):
        bad_b = lora_b.clone()
        bad_b[1, 7, rank - 1] = bad_b[1, N - 1, 0] = value
        got = tk.linear_lora(x, w, b, lora_a, bad_b, adapter, scaling)
        assert not got[mine][:, [7, N - 1]].isfinite().any()
        got[mine.nonzero(), torch.tensor([7, N - 1], device=DEV)] = clean[mine.nonzero(), torch.tensor([7, N - 1], device=DEV)]
        assert torch.equal(got, clean)
        bad_a = lora_a.clone()
        bad_a[1, rank - 1, K - 1] = value
        got = tk.linear_lora(x, w, b, bad_a, lora_b, adapter, scaling)
        assert torch.equal(got[~mine], clean[~mine]) and not got[mine].isfinite().any()
        bad_x = x.clone()
        bad_x[1, 3] = value
        got = tk.linear_lora(bad_x, w, b, lora_a, lora_b, adapter, scaling)
        assert torch.equal(got[2:], clean[2:]) and torch.equal(got[0], clean[0])
        unused = lora_a.clone(), lora_b.clone()
        unused[0][3], unused[1][3] = value, value
        others = torch.where(adapter == 3, -1, adapter)
        assert torch.equal(tk.linear_lora(x, w, b, *unused, others, scaling), tk.linear_lora(x, w, b, lora_a, lora_b, others, scaling))


@pytest.mark.gpu
def test_strides_and_empty_calls():
    g, x, w, b, lora_a, lora_b, scaling = make(1, (4, 30), 256, 200, 3, 16)
    adapter = torch.tensor([0, 2, -1, 1], device=DEV)
    check(x[:, 5:], w, b, lora_a, lora_b, adapter, scaling)                                    # a slice of longer sequences
    check(x.transpose(0, 1).contiguous().transpose(0, 1), w, b, lora_a, lora_b, adapter, scaling)
    check(x[..., 8:136], w[:, 8:136], b, lora_a[..., 8:136], lora_b, adapter, scaling)           # columns of wider operands
    check(x[..., 1:129], w[:, 1:129], b, lora_a[..., 1:129], lora_b, adapter, scaling)           # at odd addresses
    check(x, w.T.contiguous().T, b.float(), lora_a, lora_b.transpose(1, 2).contiguous().transpose(1, 2), adapter.flip(0)[::1], scaling.double())
    check(x[0, :1].expand(30, 256), w, b, lora_a, lora_b, torch.arange(30, device=DEV) % 3, scaling)
    odd = torch.empty(lora_b.numel() + 1, dtype=BF, device=DEV)[1:].view_as(lora_b).copy_(lora_b)
    check(x, w, b, lora_a, odd, adapter, scaling)
    for shape, n in (((0, 30, 256), 0), ((4, 0, 256), 4)):
        y = tk.linear_lora(torch.empty(shape, dtype=BF, device=DEV), w, b, lora_a, lora_b, torch.zeros(n, dtype=torch.int32, device=DEV), scaling)
        assert y.shape == (*shape[:-1], 200)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(6, 1024, 640), (64, 16384, 2048), (2304, 512, 2048)])
def test_the_same_bits_again_on_another_stream_and_from_graphs(M, K, N):
    g, x, w, b, lora_a, lora_b, scaling = make(M, (M,), K, N, 4, 16)
    adapter = torch.randint(-1, 4, (M,), generator=g).sort().values.to(DEV)
    call = lambda: tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, again)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append((call(), call()))
    for i in range(3):
        x.copy_(randn(g, M, K, dtype=BF))
        adapter.copy_(torch.randint(-1, 4, (M,), generator=g))
        for graph in graphs:
            graph.replay()
        eager = call()
        assert all(torch.equal(o, eager) for pair in outs for o in pair)
        torch.cuda.synchronize()


def test_the_launch_hook_sees_the_call_and_refusals_need_no_gpu(monkeypatch):
    x, w = torch.zeros(2, 3, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    a, b, i = torch.zeros(4, 2, 16, dtype=BF), torch.zeros(4, 8, 2, dtype=BF), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.linear_lora(x, w, None, a, b, i)
    with pytest.raises(KeyError):
        tk.linear_lora(x.float(), w.float(), None, a.float(), b.float(), i)
    with pytest.raises(KeyError):
        tk.linear_lora(x, w, None, a, b, i, activation="RELU")
    for bad in ((x[..., :8], w, None, a, b, i), (x, w.float(), None, a, b, i), (x, w, None, a.float(), b, i)):
        with pytest.raises(AssertionError):
            tk.linear_lora(*bad)
    monkeypatch.setattr(nv, "require_gpu", lambda *t: t[0].device)
    for bad in ((a[..., :8], b, i, None), (a, b[:, :7], i, None), (a, b[..., :1], i, None), (a[:3], b, i, None), (a, b, i[:1], None), (a, b, torch.zeros(3, dtype=torch.int32), None),
                (a, b, torch.zeros(2, 3, 16, dtype=torch.int32), None), (a, b, i, torch.zeros(3))):
        with pytest.raises(AssertionError):
            tk.linear_lora(x, w, None, *bad)
    with pytest.raises(TypeError):
        tk.linear_lora(x, w, None, a, b, i.float())
    got = tk.linear_lora_torch(x + 1, w + 1, None, a + 1, b + 1, torch.tensor([1, -1]), torch.full((4,), 0.5))
    assert torch.equal(got, torch.tensor([16 + 0.5 * 32, 16.0])[:, None, None].expand(2, 3, 8).to(BF))


@pytest.mark.gpu
def test_refusals_and_launch_hook():
    import importlib

    g, x, w, b, lora_a, lora_b, scaling = make(3, (4, 6), 64, 48, 2, 8)
    adapter = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="rank"):
        tk.linear_lora(x, w, b, torch.zeros(1, 257, 64, dtype=BF, device=DEV), torch.zeros(1, 48, 257, dtype=BF, device=DEV), adapter)
    with pytest.raises(ValueError, match="adapters"):
        tk.linear_lora(x, w, b, lora_a[:0], lora_b[:0], adapter)
    with pytest.raises(RuntimeError, match="different devices|GPU"):
        tk.linear_lora(x, w, b, lora_a, lora_b, adapter.cpu())
    linear, seen = importlib.import_module("triton_kernels.kernels.linear"), []
    linear.launch_hook = seen.append
    try:
        tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling, "GELU")
    finally:
        linear.launch_hook = None
    assert len(seen) == 1 and seen[0]["flops16"] == 2.0 * 24 * (64 * 48 + 8 * (64 + 48)) and "M=24" in seen[0]["name"]


@pytest.mark.gpu
@pytest.mark.parametrize("M,rank", [(4081, 64), (4096, 256), (4700, 33), (4609, 32), (8200, 16), (8225, 72)])
def test_first_launch_of_large_tiles(M, rank):
    """Rows enough for tiles of 32, in every count of workgroups: adapters mixed by row, in stretches that end inside a tile, and one for all."""
    g, x, w, b, lora_a, lora_b, scaling = make(M, (M,), 192, 136, 40, rank)
    for adapter in (torch.randint(-1, 40, (M,), generator=g), torch.arange(M) // 37 % 41 - 1, torch.randint(0, 40, (), generator=g)):
        check(x, w, b, lora_a, lora_b, adapter.to(DEV), scaling)
    check(x[:M // 7 * 7].view(-1, 7, 192), w, b, lora_a, lora_b, torch.randint(-1, 40, (M // 7,), generator=g).to(DEV), scaling)
