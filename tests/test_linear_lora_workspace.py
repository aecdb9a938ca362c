"""linear_lora's workspace: what lay in it before a call reaches no result, and graphs that were captured with it replay the eager results."""
import ctypes

import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from test_linear_lora import make
from util import DEV, randn

BF = torch.bfloat16
SHAPES = [(5, 512, 384), (9, 256, 64), (33, 512, 520), (64, 16384, 2048), (300, 256, 520), (517, 2048, 2048), (2305, 512, 1536), (4099, 512, 4096), (20, 63, 50)]


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [3, 16, 17, 40, 72])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_what_lay_there_before(M, K, N, rank):
    """Memory full of NaN and of infinities: rows without an adapter, rows behind the last, places behind the rank."""
    g, x, w, b, lora_a, lora_b, scaling = make(M + rank, (M,), K, N, 3, rank)
    lib = nv.lib()
    for owner in (torch.randint(-1, 3, (M,), generator=g, dtype=torch.int32).to(DEV), (torch.arange(M) // 9 % 4 - 1).int().to(DEV)):
        want = tk.linear_lora(x, w, b, lora_a, lora_b, owner, scaling)
        assert want.isfinite().all()
        y = torch.empty_like(want)
        args = nv.LinearLoraArgs(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), owner.data_ptr(), scaling.data_ptr(), M, N, K, K, K, N, M, 3, rank, 0, 0)
        need = lib.flux_linear_lora_workspace_bytes(ctypes.byref(args))
        for fill in (-1, 0x7F807F80):
            ws = torch.full(((need + 4096) // 4,), fill, dtype=torch.int32, device=DEV)
            assert lib.flux_linear_lora_bf16(ctypes.byref(args), ws.data_ptr(), need, nv.stream_ptr(x.device)) == 0
            assert torch.equal(y, want) and (ws[need // 4:] == fill).all()
        least = lib.flux_linear_lora_least_bytes(ctypes.byref(args))
        ws = torch.full(((least + 4096) // 4,), -1, dtype=torch.int32, device=DEV)
        assert lib.flux_linear_lora_bf16(ctypes.byref(args), ws.data_ptr(), least, nv.stream_ptr(x.device)) == 0
        assert y.isfinite().all() and (ws[least // 4:] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,rank", [(6, 1024, 640, 40), (64, 16384, 2048, 40), (517, 512, 2048, 32), (2304, 512, 2048, 72)])
def test_two_graphs_between_eager_calls(M, K, N, rank):
    g, x, w, b, lora_a, lora_b, scaling = make(M, (M,), K, N, 4, rank)
    adapter = torch.randint(-1, 4, (M,), generator=g).to(DEV)
    call = lambda: tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling)  # noqa: E731
    call()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph, pool=graphs[0].pool() if outs else None):
            outs.append((call(), call()))
    for _ in range(3):
        x.copy_(randn(g, M, K, dtype=BF))
        adapter.copy_(torch.randint(-1, 4, (M,), generator=g))
        eager = call()
        for graph, pair in zip(graphs, outs):
            graph.replay()
            assert all(torch.equal(o, eager) for o in pair)
        torch.cuda.synchronize()
