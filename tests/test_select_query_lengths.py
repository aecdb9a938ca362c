"""Selection of blocks for padded queries: rows behind a sequence's end have no share in the lists of those in front of it."""
import ctypes
import math

import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from test_select_blocks import expected, inputs
from test_tune_native_calls import launcher, took
from util import DEV, seeded


def padded(q, k, keep, always, lengths, ends):
    """Each sequence by itself, cut at its ends; -1 for blocks behind them."""
    out = torch.full((q.shape[0], q.shape[1], -(-q.shape[2] // 128), min(keep, -(-k.shape[2] // 64))), -1, dtype=torch.int32)
    for b in range(q.shape[0]):
        n, m = (min(max(int(t[b]), 0), most) for t, most in ((ends, q.shape[2]), (lengths, k.shape[2])))
        if n and m:
            one = expected(q[b:b + 1, :, :n], k[b:b + 1, :, :m], keep, always)
            out[b, :, :one.shape[2], :one.shape[3]] = one[0]
    return out


SHAPES = [(2, 4, 2, 300, 300, 64, 3, 1, [300, 150], [300, 150]), (3, 2, 1, 1084, 1084, 128, 5, 0, [1084, 1, 129], [1084, 1, 129]), (4, 2, 2, 700, 2000, 64, 7, 2, [700, 0, 128, 256], [2000, 1500, 64, 900]),
          (2, 1, 1, 257, 64 * 1030, 64, 20, 3, [130, 256], [66000, 64 * 1030]), (2, 2, 1, 130, 150, 128, 9, 0, [129, 7], [150, 40]), (3, 1, 1, 2300, 1000, 64, 4, 1, [2300, 2049, 100], [1000, 900, 0])]


@pytest.mark.parametrize("B,Hq,Hk,Lq,Lk,D,keep,always,ends,lengths", SHAPES)
def test_the_plain_statement(B, Hq, Hk, Lq, Lk, D, keep, always, ends, lengths):
    q, k = inputs(seeded(Lq), B, Hq, Hk, Lq, Lk, D)
    want = padded(q, k, keep, always, lengths, ends)
    for b, n in enumerate(ends):
        q[b, :, n:] = math.nan
    assert torch.equal(tk.select_blocks_torch(q, k, keep, always, torch.tensor(lengths), torch.tensor(ends)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hq,Hk,Lq,Lk,D,keep,always,ends,lengths", SHAPES)
def test_what_stands_behind_the_queries_does_not_matter(B, Hq, Hk, Lq, Lk, D, keep, always, ends, lengths):
    q, k = inputs(seeded(Lq), B, Hq, Hk, Lq, Lk, D)
    want = padded(q, k, keep, always, lengths, ends)
    ends_, lengths_ = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in (ends, lengths))
    for fill in (0.0, 100.0, math.inf, math.nan):
        for b, n in enumerate(ends):
            q[b, :, n:] = fill
        assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), keep, always=always, lengths=lengths_, q_lengths=ends_).cpu(), want)
    # other whole types, numbers below 0 and beyond the rows
    far = torch.tensor([e if e < Lq and e > 0 else (2 ** 33 if e else -5) for e in ends], device=DEV)
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), keep, always=always, lengths=lengths_, q_lengths=far).cpu(), want)


@pytest.mark.gpu
def test_without_them_all_rows_are_queries():
    q, k = inputs(seeded(1), 2, 2, 2, 300, 640, 64)
    whole = torch.full((2,), 300, dtype=torch.int32, device=DEV)
    want = expected(q, k, 4)
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 4).cpu(), want) and torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 4, q_lengths=whole).cpu(), want)


@pytest.mark.gpu
def test_a_padded_batch_that_attends_to_itself():
    """Selection and attention one behind the other: real rows are those of each sequence by itself, rows of blocks behind a sequence are 0."""
    g = seeded(2)
    q, k = inputs(g, 2, 4, 2, 500, 500, 128)
    v = inputs(g, 2, 4, 2, 500, 500, 128)[1]
    ends = [500, 201]
    for b, n in enumerate(ends):
        for t in (q, k, v):
            t[b, :, n:] = math.nan
    q, k, v, lengths = q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(ends, dtype=torch.int32, device=DEV)
    blocks = tk.select_blocks(q, k, 3, lengths=lengths, q_lengths=lengths)
    o = tk.block_sparse_attention(q, k, v, blocks, lengths=lengths)
    for b, n in enumerate(ends):
        alone = [t[b:b + 1, :, :n] for t in (q, k, v)]
        lists = tk.select_blocks(*alone[:2], 3)
        assert torch.equal(blocks[b, :, :-(-n // 128)], lists[0])
        assert torch.equal(o[b, :, :n], tk.block_sparse_attention(*alone, lists)[0])
    assert bool((o[1, :, 256:] == 0).all())


@pytest.mark.gpu
def test_lengths_that_change_between_replays():
    g = seeded(3)
    q, k = (t.to(DEV) for t in inputs(g, 2, 2, 1, 400, 700, 64))
    ends = torch.tensor([400, 400], dtype=torch.int32, device=DEV)
    tk.select_blocks(q, k, 3, q_lengths=ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tk.select_blocks(q, k, 3, q_lengths=ends)
    for pair in ([400, 1], [0, 130], [129, 399], [400, 400]):
        ends.copy_(torch.tensor(pair, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), padded(q.cpu(), k.cpu(), 3, 0, [700, 700], pair))


@pytest.mark.gpu
def test_refusals_of_a_call():
    q, k = (torch.zeros(2, 2, 100, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    with pytest.raises(AssertionError):
        tk.select_blocks(q, k, 1, q_lengths=torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        tk.select_blocks(q, k, 1, q_lengths=torch.zeros(2, device=DEV))
    with pytest.raises(RuntimeError):
        tk.select_blocks(q, k, 1, q_lengths=torch.zeros(2, dtype=torch.int32))


def test_the_structure_ends_with_them():
    """Programs that fill the fields in front of it by position leave it null."""
    assert nv.SelectBlocksArgs._fields_[-1][0] == "q_lengths" and nv.SelectBlocksArgs(D=64).q_lengths is None
    assert nv.SelectBlocksArgs.q_lengths.offset == ctypes.sizeof(nv.SelectBlocksArgs) - 8


@pytest.mark.gpu
def test_native_call_and_launcher(monkeypatch):
    q, k = (t.to(DEV) for t in inputs(seeded(4), 2, 4, 2, 300, 500, 64))
    ends, lengths = torch.tensor([300, 70], dtype=torch.int32, device=DEV), torch.tensor([130, 500], dtype=torch.int32, device=DEV)
    for kw in (dict(q_lengths=ends), dict(q_lengths=ends, lengths=lengths, always=1)):
        assert took(monkeypatch, tk.select_blocks, q, k, 3, **kw)
        assert torch.equal(tk.select_blocks(q, k, 3, **kw), launcher(monkeypatch, tk.select_blocks, q, k, 3, **kw))
    for other in (ends.long(), ends.repeat_interleave(2)[::2]):
        assert not took(monkeypatch, tk.select_blocks, q, k, 3, q_lengths=other)
        assert torch.equal(tk.select_blocks(q, k, 3, q_lengths=other), tk.select_blocks(q, k, 3, q_lengths=ends))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_from_code_that_is_traced(backend):
    torch._dynamo.reset()
    q, k = (t.to(DEV) for t in inputs(seeded(5), 2, 2, 2, 300, 300, 64))
    ends = torch.tensor([300, 70], dtype=torch.int32, device=DEV)
    fn = lambda q: tk.select_blocks(q * 1.0, k, 2, lengths=ends, q_lengths=ends) + 0  # noqa: E731
    assert torch.equal(torch.compile(fn, backend=backend)(q), fn(q))
    torch._dynamo.reset()


@pytest.mark.gpu
def test_two_streams_and_two_graphs_of_one_pool():
    g = seeded(6)
    q, k = (t.to(DEV) for t in inputs(g, 2, 2, 1, 700, 64 * 40, 64))
    far = inputs(g, 2, 2, 1, 700, 64 * 1030, 64)[1].to(DEV)   # (scores in the workspace)
    ends = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([700, 130], [257, 0])]
    calls = [lambda e=e, t=t: tk.select_blocks(q, t, 9, q_lengths=e) for e in ends for t in (k, far)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append([c() for c in calls])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for each in got for a, b in zip(each, want))
    pool, graphs, outs = None, [], []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(c())
        pool = graph.pool()
        graphs.append(graph)
    for _ in range(3):
        for graph, out, expected_ in zip(graphs, outs, want):
            graph.replay()
            assert torch.equal(out, expected_)
