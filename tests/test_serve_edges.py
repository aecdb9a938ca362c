"""Calls of linear_w4, select_blocks and block_sparse_attention at the edges of what they take."""
import sys

import pytest
import torch

import triton_kernels as tk
from triton_kernels.kernels import attention as attention_calls
from triton_kernels.modules import LinearW4, Modulation
from util import DEV, randn, seeded

BF = torch.bfloat16
WHOLE = [torch.uint8, torch.int8, torch.int16, torch.int64, torch.uint16, torch.uint32, torch.uint64]


@pytest.mark.parametrize("dtype", WHOLE)
def test_lengths_of_every_whole_type(dtype):
    lengths = torch.tensor([5, 100], dtype=torch.int64).to(dtype)
    got = attention_calls._lengths(lengths, 2, lengths.device, 4608)
    assert got.dtype == torch.int32 and got.tolist() == [5, 100]
    long = torch.tensor([-3, 2 ** 40])
    assert attention_calls._lengths(long, 2, long.device, 70).tolist() == [0, 70]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", WHOLE)
def test_lists_and_lengths_of_every_whole_type(dtype):
    g = seeded(1)
    q, k, v = (randn(g, 2, h, 200, 64, dtype=BF).to(DEV) for h in (4, 2, 2))
    blocks, lengths = torch.randint(0, 5, (2, 4, 2, 3), generator=g).to(DEV), torch.tensor([127, 70], device=DEV)
    want = tk.block_sparse_attention(q, k, v, blocks.int(), lengths=lengths.int()), tk.select_blocks(q, k, 2, lengths=lengths.int())
    assert torch.equal(tk.block_sparse_attention(q, k, v, blocks.to(dtype), lengths=lengths.to(dtype)), want[0])
    assert torch.equal(tk.select_blocks(q, k, 2, lengths=lengths.to(dtype)), want[1])


@pytest.mark.gpu
def test_counts_beyond_64_bits():
    g = seeded(2)
    q, k = (randn(g, 1, 2, 300, 64, dtype=BF).to(DEV) for _ in range(2))
    every = torch.arange(5, dtype=torch.int32, device=DEV).expand(1, 2, 3, 5)
    for keep in (2 ** 64, 2 ** 65 + 1, 2 ** 62, 5):
        assert torch.equal(tk.select_blocks(q, k, keep), every)
        assert torch.equal(tk.select_blocks(q, k, 3, always=keep), every[..., :3])


def test_quantised_weights_of_the_whole_range():
    w = torch.tensor([[-3e38, 3e38, 0.0, 1e38] * 8, [1e-30, -1e-30, 0.0, 5e-31] * 8, [3e38] * 32])
    for zeros in (False, True):
        q, scale, zero = tk.quantize_w4(w, 32, zeros).unpack()
        assert bool(scale.isfinite().all()) and bool((scale > 0).all())
        back = (q.double() - (8.0 if zero is None else zero.double().repeat_interleave(32, 1))) * scale.double().repeat_interleave(32, 1)
        # half a step each for the value and the zero point, and half a bf16 step of the scale for 15 of them
        assert bool(((back - w.double()).abs() <= scale.double().repeat_interleave(32, 1) * (1.0 + 15 * 2.0 ** -8)).all())


def test_a_weight_is_quantised_once():
    m = Modulation(64, double=False).quantize(32, True)
    before = m.lin.weight.unpack()
    with pytest.raises(AssertionError, match="LinearW4"):
        m.quantize()
    assert isinstance(m.lin, LinearW4) and all(torch.equal(a, b) for a, b in zip(before, m.lin.weight.unpack()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 129])
def test_a_hook_hears_of_the_product(monkeypatch, rows):
    module, heard = sys.modules["triton_kernels.kernels.linear"], []   # (the package's attribute of that name is the function)
    g = seeded(rows)
    w, x = tk.quantize_w4(randn(g, 17, 96), 32).to(DEV), randn(g, rows, 96, dtype=BF).to(DEV)
    want = tk.linear_w4(x, w)
    monkeypatch.setattr(module, "launch_hook", heard.append)
    assert torch.equal(tk.linear_w4(x, w, in_activation="SiLU" if rows == 1 else ""), want) == (rows > 1)
    assert len(heard) == 1 and heard[0]["flops16"] == 2 * rows * 17 * 96 and heard[0]["bytes"] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 128, 129, 300])
def test_rows_that_are_one_row(rows):
    """An expanded row, odd numbers of outputs and the shortest rows there are, also where the weights are laid out first."""
    g = seeded(rows)
    w, x = tk.quantize_w4(randn(g, 17, 32), 32).to(DEV), randn(g, 1, 32, dtype=BF).to(DEV)
    y = tk.linear_w4(x.expand(rows, 32), w)
    assert torch.equal(y, tk.linear_w4(x.repeat(rows, 1), w)) and torch.equal(y, y[:1].expand(rows, 17))
    # weights rounded to bf16 beyond 128 rows, the result to bf16; fp32 sums of 32 terms of up to 31 |x| s, with and without the weight
    q, scale, _ = w.to("cpu").unpack()
    wf = (q.double() - 8) * scale.double().repeat_interleave(32, 1)
    want, size = x.double().cpu() @ wf.T, x.double().abs().cpu() @ wf.abs().T
    sums = x.double().abs().cpu().sum() * scale.double().T * 31 * 2 * 32 * 2.0 ** -24
    off = (want.abs() * 2.0 ** -8 + size * (2.0 ** -8 if rows > 128 else 0.0) + sums) * 1.01
    assert bool(((y[:1].double().cpu() - want).abs() <= off).all())


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_calls_from_code_that_is_traced(backend):
    torch._dynamo.reset()
    g = seeded(3)
    w, x = tk.quantize_w4(randn(g, 40, 64), 64).to(DEV), randn(g, 3, 64, dtype=BF).to(DEV)
    q, k = randn(g, 1, 2, 300, 64, dtype=BF).to(DEV), randn(g, 1, 2, 300, 64, dtype=BF).to(DEV)
    blocks = tk.select_blocks(q, k, 2)
    for fn, args in ((lambda x: tk.linear_w4(x * 1.0, w, activation="GELU") * 2.0, (x,)), (lambda q, k: tk.select_blocks(q * 1.0, k, 2, always=1) + 0, (q, k)),
                     (lambda q, k: tk.block_sparse_attention(q * 1.0, k, k, blocks, 0.1) * 1.0, (q, k)), (lambda q, k: tk.block_sparse_attention(q, k, k, tk.select_blocks(q, k, 3)) * 1.0, (q, k))):
        assert torch.equal(torch.compile(fn, backend=backend)(*args), fn(*args))
        torch._dynamo.reset()   # (what was compiled for it before serves a second call too)
        with pytest.raises(Exception):
            torch.compile(fn, backend=backend, fullgraph=True)(*args)
    torch._dynamo.reset()


@pytest.mark.gpu
def test_two_operators_at_once_on_two_streams():
    """The same operands on two streams, each call with a workspace of its own."""
    g = seeded(4)
    w, x = tk.quantize_w4(randn(g, 256, 512), 128).to(DEV), randn(g, 200, 512, dtype=BF).to(DEV)
    q, k = randn(g, 1, 2, 70, 128, dtype=BF).to(DEV), randn(g, 1, 2, 64 * 40, 128, dtype=BF).to(DEV)
    far, far_k = q[..., :64].contiguous(), randn(g, 1, 2, 64 * 1030, 64, dtype=BF).to(DEV)

    def calls():
        blocks = tk.select_blocks(q, k, 30)
        return tk.linear_w4(x, w), blocks, tk.block_sparse_attention(q, k, k, blocks), tk.select_blocks(far, far_k, 9)

    want, streams = calls(), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for each in got for a, b in zip(each, want))


def _args(M, N, K, ldx):
    from triton_kernels import _native as nv
    return nv.LinearW4Args(256, None, 256, nv.W4(256, 256, None, N, K, 64), M, ldx, N, 0, 0)


def test_workspaces_of_products():
    """Up to 128 rows, and for hundreds of rows of thousands of outputs, none; else room for the weights in bf16."""
    from triton_kernels import _native as nv
    need = lambda *a: nv.lib().flux_linear_w4_workspace_bytes(nv.byref(_args(*a)))  # noqa: E731
    assert [need(128, 9216, 3072, 3072), need(256, 9216, 3072, 3072), need(512, 9216, 3072, 4096), need(0, 9216, 3072, 3072)] == [0] * 4
    for M, N, K, ldx in ((129, 4608, 64, 64), (256, 3072, 3072, 3072), (4096, 9216, 3072, 3072), (256, 9216, 64, 2 ** 23)):
        assert need(M, N, K, ldx) >= N * K * 2


@pytest.mark.gpu
def test_rows_that_lie_far_apart():
    g = seeded(6)
    w, rows = tk.quantize_w4(randn(g, 9216, 64), 64).to(DEV), randn(g, 130, 64, dtype=BF).to(DEV)
    x = torch.empty(129 * 2 ** 23 + 64, dtype=BF, device=DEV).as_strided((130, 64), (2 ** 23, 1))
    x.copy_(rows)
    y, near = tk.linear_w4(x, w), tk.linear_w4(rows, w)
    wf = w.dequantize().double()   # (rounded; both ways sum 64 products of it and round once)
    want, size = rows.double() @ wf.t(), rows.double().abs() @ wf.abs().t()
    for got in (y, near):
        assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2 * 64 * 2.0 ** -24).all())
    assert torch.equal(tk.linear_w4(x[:128], w), tk.linear_w4(rows[:128], w))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_modules_in_code_that_is_traced(backend):
    torch._dynamo.reset()
    g = seeded(7)
    lin = torch.nn.Linear(128, 80)
    lin.weight.data, lin.bias.data = randn(g, 80, 128), randn(g, 80)
    served = LinearW4.from_linear(lin, 64, True).to(DEV)
    mod = Modulation(128, double=False)
    mod.lin.weight.data, mod.lin.bias.data = randn(g, 384, 128), randn(g, 384)
    mod = mod.bfloat16().quantize(32).to(DEV)
    x = randn(g, 3, 128, dtype=BF).to(DEV)
    with torch.no_grad():
        assert torch.equal(torch.compile(served, backend=backend)(x * 2.0), served(x * 2.0))
        got, want = torch.compile(mod, backend=backend)(x)[0], mod(x)[0]
        assert torch.equal(got.scale, want.scale) and torch.equal(got.shift, want.shift) and torch.equal(got.gate, want.gate)
    torch._dynamo.reset()


@pytest.mark.gpu
def test_lengths_that_change_between_replays():
    g = seeded(8)
    q, k, v = (randn(g, 2, h, 700, 64, dtype=BF).to(DEV) for h in (4, 2, 2))
    lengths = torch.tensor([700, 700], dtype=torch.int32, device=DEV)

    def calls(of):
        blocks = tk.select_blocks(q, k, 3, always=1, lengths=of)
        return blocks, tk.block_sparse_attention(q, k, v, blocks, lengths=of)

    calls(lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls(lengths)
    for pair in ([700, 1], [0, 130], [64, 699], [700, 700]):
        lengths.copy_(torch.tensor(pair, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = calls(torch.tensor(pair, dtype=torch.int32, device=DEV))
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_under_autocast_and_inference_mode():
    g = seeded(9)
    w, x = tk.quantize_w4(randn(g, 40, 64), 32).to(DEV), randn(g, 3, 64, dtype=BF).to(DEV)
    q = randn(g, 1, 2, 300, 128, dtype=BF).to(DEV)
    want = tk.linear_w4(x, w), tk.select_blocks(q, q, 2), tk.block_sparse_attention(q, q, q, tk.select_blocks(q, q, 2))
    for mode in (torch.inference_mode(), torch.autocast("cuda", dtype=torch.float16), torch.autocast("cuda", dtype=BF)):
        with mode:
            got = tk.linear_w4(x, w), tk.select_blocks(q, q, 2), tk.block_sparse_attention(q, q, q, tk.select_blocks(q, q, 2))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
