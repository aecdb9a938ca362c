"""Attention over listed blocks of keys against the formula in float64 on the CPU, what is not listed, and what is refused."""
import ctypes
import math

import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded

HALF = torch.finfo(torch.bfloat16).eps / 2


def expected(q, k, v, blocks, scale=None, lengths=None):
    """The result in float64, how far a value may be from it, and the root mean square of all differences that independent roundings leave.

    q times the scale is off by half a step a value, which moves a score by at most HALF sum |q k| and, roundings being spread evenly, by HALF / sqrt(3) times
    the root of the sum of the squares; probabilities and result are off by half a step each. Sums in fp32 add (64 tiles of) 2^-23 of what they sum."""
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    count = -(-Lk // 64)
    out, off, mean = (torch.zeros(B, Hq, Lq, D, dtype=torch.float64) for _ in range(3))
    for b in range(B):
        end = Lk if lengths is None else min(max(int(lengths[b]), 0), Lk)
        for h in range(Hq):
            kh, vh = k[b, h // (Hq // Hk)].double(), v[b, h // (Hq // Hk)].double()
            for t in range(-(-Lq // 128)):
                names = [j for j in blocks[b, h, t].tolist() if 0 <= j < count]
                tokens = torch.tensor([i for j in names for i in range(j * 64, min(j * 64 + 64, end))], dtype=torch.long)
                rows = slice(t * 128, min(t * 128 + 128, Lq))
                if len(tokens) == 0:
                    continue
                qt, kt, vt = q[b, h, rows].double(), kh[tokens], vh[tokens]
                p = torch.softmax(qt @ kt.T * scale, -1)
                o = p @ vt
                moved = HALF * (qt.abs() @ kt.abs().T) * abs(scale)
                spread = HALF / 3 ** 0.5 * ((qt ** 2) @ (kt ** 2).T).sqrt() * abs(scale)
                worst = moved.amax(-1, keepdim=True)
                reach = p @ vt.abs()
                err = (torch.exp(2 * worst) - 1 + HALF + 2.0 ** -16) * (reach + o.abs())
                out[b, h, rows], off[b, h, rows] = o, err + HALF * (o.abs() + err)
                mean[b, h, rows] = ((p ** 2 * (spread ** 2 + HALF ** 2 / 3)) @ vt ** 2 + o ** 2 * (((p * spread) ** 2).sum(-1, keepdim=True) + HALF ** 2 / 3)).sqrt()
    return out, off, mean


def check(got, q, k, v, blocks, scale=None, lengths=None):
    want, off, mean = expected(q.cpu(), k.cpu(), v.cpu(), blocks.cpu(), scale, lengths)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= off).all()), f"{(err - off).max().item():.3e} beyond the bound"
    # scores' errors of neighbouring keys go together in part, and outliers weigh: one and a half times what independent ones leave
    assert err.pow(2).mean().sqrt() <= 1.5 * mean.pow(2).mean().sqrt() + 1e-30


def inputs(g, B, Hq, Hk, Lq, Lk, D, std=1.0):
    q = randn(g, B, Lq, Hq, D, dtype=torch.bfloat16, std=std).transpose(1, 2)
    k, v = (randn(g, B, Lk, Hk, D, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    return q, k, v


def lists(g, B, Hq, Lq, Lk, count, some=False):
    """Lists of different blocks in any order; `some`: a third of the entries name nothing."""
    have = -(-Lk // 64)
    b = torch.stack([torch.randperm(have, generator=g)[:count] for _ in range(B * Hq * -(-Lq // 128))]).view(B, Hq, -1, min(count, have)).to(torch.int32)
    if some:
        b[torch.rand(b.shape, generator=g) < 0.33] = -1
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hq,Hk,Lq,Lk,D,count,some,padded", [
    (1, 1, 1, 1, 1, 128, 1, False, False), (1, 1, 1, 1, 1, 64, 1, False, False), (1, 2, 1, 128, 64, 64, 1, False, False), (2, 4, 2, 129, 65, 128, 2, False, True), (1, 3, 3, 300, 640, 64, 3, True, False),
    (2, 2, 2, 1084, 1084, 128, 5, True, True), (3, 4, 1, 1, 2000, 64, 7, False, True), (3, 6, 2, 5, 2001, 128, 31, True, True), (1, 1, 1, 200, 8200, 64, 129, False, False), (1, 1, 1, 130, 8200, 128, 129, True, False),
    (1, 2, 2, 127, 4160, 128, 64, False, False), (1, 2, 2, 127, 4160, 64, 65, True, True), (1, 24, 8, 1, 3000, 128, 40, False, False), (1, 1, 1, 260, 100, 128, 2, False, False)])
def test_against_float64(B, Hq, Hk, Lq, Lk, D, count, some, padded):
    g = seeded(Lq * 7 + Lk)
    q, k, v = inputs(g, B, Hq, Hk, Lq, Lk, D)
    blocks = lists(g, B, Hq, Lq, Lk, count, some)
    lengths = torch.tensor([Lk, max(Lk // 3, 1), 0][:B], dtype=torch.int32) if padded else None
    got = tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV), lengths=None if lengths is None else lengths.to(DEV))
    assert got.shape == q.shape and got.is_contiguous()
    check(got, q, k, v, blocks, None, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("std,scale", [(4.0, None), (1.0, -0.2), (1.0, 0.0), (0.01, 30.0)])
def test_scores_of_other_sizes(std, scale):
    g = seeded(6)
    q, k, v = inputs(g, 1, 2, 1, 300, 700, 128, std)
    blocks = lists(g, 1, 2, 300, 700, 6)
    check(tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV), scale), q, k, v, blocks, scale)


@pytest.mark.gpu
def test_every_block_is_attention_over_all_keys():
    g = seeded(7)
    q, k, v = (t.to(DEV) for t in inputs(g, 2, 3, 3, 450, 450, 128))
    every = torch.arange(8, dtype=torch.int32, device=DEV).expand(2, 3, 4, 8)
    dense = tk.scaled_dot_product_attention(q, k, v)
    # two roundings of the same sums, one of them of the probabilities' sum as well
    assert (tk.block_sparse_attention(q, k, v, every).double() - dense.double()).abs().max() <= 4 * HALF * dense.abs().max()
    check(tk.block_sparse_attention(q, k, v, every), q, k, v, every)


@pytest.mark.gpu
def test_what_is_not_listed_or_behind_the_length_does_not_matter():
    g = seeded(8)
    q, k, v = inputs(g, 2, 2, 2, 200, 500, 64)
    blocks = torch.tensor([[5, 1], [7, 3]], dtype=torch.int32).expand(2, 2, 2, 2).contiguous()
    lengths = torch.tensor([350, 480])
    want = tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV), lengths=lengths.to(DEV))
    check(want, q, k, v, blocks, None, lengths)
    for b, n in enumerate(lengths.tolist()):
        for t in (k, v):
            t[b, :, n:] = math.nan
            for j in (0, 2, 4, 6):
                t[b, :, j * 64:j * 64 + 64] = math.inf if j % 4 else math.nan
    for kind in (torch.int32, torch.int64):
        assert torch.equal(tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV, kind), lengths=lengths.to(DEV, kind)), want)


@pytest.mark.gpu
def test_lists_that_name_nothing():
    g = seeded(9)
    q, k, v = (t.to(DEV) for t in inputs(g, 2, 2, 1, 300, 200, 128))
    none = torch.full((2, 2, 3, 4), -1, dtype=torch.int32, device=DEV)
    assert bool((tk.block_sparse_attention(q, k, v, none) == 0).all())
    assert bool((tk.block_sparse_attention(q, k, v, none[..., :0]) == 0).all())
    assert bool((tk.block_sparse_attention(q, k[:, :, :0], v[:, :, :0], none) == 0).all())
    far = none.long()
    far[..., 0], far[..., 1], far[..., 2], far[..., 3] = 4, 2 ** 32, -2 ** 31, 2 ** 31 + 1   # none of them a block of 200 keys
    assert bool((tk.block_sparse_attention(q, k, v, far) == 0).all())
    assert bool((tk.block_sparse_attention(q, k, v, far.clamp(-2 ** 31, 2 ** 31 - 1).int()) == 0).all())
    lists_ = none.clone()
    lists_[:, :, 1] = torch.tensor([-1, 3, -1, 0], dtype=torch.int32)
    got = tk.block_sparse_attention(q, k, v, lists_)
    assert bool((got[:, :, :128] == 0).all()) and bool((got[:, :, 256:] == 0).all())
    check(got, q, k, v, lists_)
    lengths = torch.tensor([0, 129], device=DEV)
    got = tk.block_sparse_attention(q, k, v, lists_, lengths=lengths)
    assert bool((got[0] == 0).all())
    check(got, q, k, v, lists_, None, lengths.tolist())


@pytest.mark.gpu
def test_order_and_repetition():
    g = seeded(10)
    q, k, v = inputs(g, 1, 1, 1, 100, 640, 128)
    a = torch.tensor([[[[9, 2, 5]]]], dtype=torch.int32)
    for order in ([2, 5, 9], [5, 9, 2], [-1, 9, 5, -1, 2, -1]):
        b = torch.tensor(order, dtype=torch.int32).view(1, 1, 1, -1)
        check(tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), b.to(DEV)), q, k, v, a)
    twice = torch.tensor([[[[9, 2, 5, 9]]]], dtype=torch.int32)
    check(tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), twice.to(DEV)), q, k, v, twice)
    one = torch.tensor([[[[4, 4, 4]]]], dtype=torch.int32)
    check(tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), one.to(DEV)), q, k, v, one[..., :1])


@pytest.mark.gpu
def test_values_that_are_not_finite():
    g = seeded(11)
    q, k, v = inputs(g, 1, 1, 1, 256, 256, 64)
    blocks = torch.tensor([[1, 2], [0, 3]], dtype=torch.int32).view(1, 1, 2, 2)
    v[0, 0, 70, 3], v[0, 0, 200, 5] = math.nan, math.inf
    q[0, 0, 9] = math.nan
    got = tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV)).cpu()
    want = expected(q, k, v, blocks)[0]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert (got[fine].double() - want[fine]).abs().max() <= 0.1


@pytest.mark.gpu
def test_views_and_a_given_result():
    g = seeded(12)
    wide = randn(g, 2, 333, 3, 4, 136, dtype=torch.bfloat16).to(DEV)
    q, k, v = wide[:, :, 0, :, :128].transpose(1, 2), wide[:, 20:, 1, :2, 8:].transpose(1, 2), wide[:, 20:, 2, 2:, :128].transpose(1, 2)
    blocks = lists(g, 2, 4, 333, 313, 3).to(DEV)
    want = tk.block_sparse_attention(q, k, v, blocks)
    check(want, q, k, v, blocks)
    odd = wide[:, 20:, 2, 2:, 1:129].transpose(1, 2)
    check(tk.block_sparse_attention(q, k, odd, blocks), q, k, odd, blocks)
    assert torch.equal(tk.block_sparse_attention(q, k, v, blocks.repeat_interleave(2, -1)[..., ::2]), want)
    held = torch.full((2, 340, 4, 144), 7.0, dtype=torch.bfloat16, device=DEV)
    out = held[:, :333, :, 8:136].transpose(1, 2)
    assert tk.block_sparse_attention(q, k, v, blocks, out=out) is out and torch.equal(out, want)
    held[:, :333, :, 8:136] = 7.0
    assert bool((held == 7.0).all())   # nothing beside it was written
    assert tk.block_sparse_attention(q[:, :, :0], k, v, blocks[:, :, :0]).shape == (2, 4, 0, 128)


@pytest.mark.gpu
def test_keys_that_lie_beyond_32_bits():
    g = seeded(13)
    k, v = (torch.empty(300, 1 << 23, dtype=torch.bfloat16, device=DEV)[:, :64] for _ in range(2))   # 2^31 values to row 256
    k.copy_(randn(g, 300, 64)), v.copy_(randn(g, 300, 64))
    q = randn(g, 1, 1, 128, 64, dtype=torch.bfloat16).to(DEV)
    blocks = torch.tensor([[[[4, 0]]]], dtype=torch.int32, device=DEV)
    check(tk.block_sparse_attention(q, k[None, None], v[None, None], blocks), q, k[None, None], v[None, None], blocks)
    assert torch.equal(tk.select_blocks(q, k[None, None], 2), tk.select_blocks(q, k[None, None].clone(memory_format=torch.contiguous_format), 2))


@pytest.mark.gpu
def test_selection_and_attention_together_on_streams_and_in_graphs():
    g = seeded(14)
    q, k, v = (t.to(DEV) for t in inputs(g, 2, 4, 2, 700, 700, 128))
    lengths = torch.tensor([700, 400], device=DEV)

    def run(q):
        blocks = tk.select_blocks(q, k, 4, always=1, lengths=lengths)
        return blocks, tk.block_sparse_attention(q, k, v, blocks, lengths=lengths)

    blocks, want = run(q)
    check(want, q, k, v, blocks, None, lengths.tolist())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = run(q)
    stream.synchronize()
    assert torch.equal(other[0], blocks) and torch.equal(other[1], want)
    mine, graph = q.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(mine)
    for _ in range(3):
        mine.copy_(randn(g, 2, 4, 700, 128, dtype=torch.bfloat16))
        graph.replay()
        again = run(mine)
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


@pytest.mark.gpu
def test_gradients_are_an_error():
    q = torch.zeros(1, 1, 8, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    k = torch.zeros(1, 1, 64, 64, dtype=torch.bfloat16, device=DEV)
    blocks = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(NotImplementedError):
        tk.block_sparse_attention(q, k, k, blocks).sum().backward()
    with pytest.raises(AssertionError):
        tk.block_sparse_attention(q, k, k, blocks, out=torch.empty_like(q))
    with torch.no_grad():
        assert not tk.block_sparse_attention(q, k, k, blocks, out=torch.empty_like(q)).requires_grad


@pytest.mark.gpu
def test_refusals_of_a_call():
    q, k = torch.zeros(2, 4, 100, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 2, 100, 64, dtype=torch.bfloat16, device=DEV)
    b = torch.zeros(2, 4, 1, 2, dtype=torch.int32, device=DEV)
    f = tk.block_sparse_attention
    for bad in (lambda: f(q[0], k, k, b), lambda: f(q, k[:1], k[:1], b), lambda: f(q[:, :3], k, k, b[:, :3]), lambda: f(q[..., :32], k[..., :32], k[..., :32], b), lambda: f(q, k, k[:, :, :99], b), lambda: f(q, k, k, b[0]),
                lambda: f(q, k, k, b[:, :2]), lambda: f(q, k, k, b.expand(2, 4, 1, 2)[:, :, :0]), lambda: f(q, k, k, b, lengths=torch.zeros(1, dtype=torch.int32, device=DEV)), lambda: f(q, k, k, b, out=q[:, :, :99]),
                lambda: f(q, k, k, b, out=torch.empty(2, 4, 64, 100, dtype=q.dtype, device=DEV).transpose(2, 3))):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: f(q.float(), k.float(), k.float(), b), lambda: f(q, k, k, b.float()), lambda: f(q, k, k, b, lengths=torch.zeros(2, device=DEV)), lambda: f(q, k, k, b, out=torch.empty_like(q, dtype=torch.float32))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        f(q, k, k.cpu(), b)
    with pytest.raises(NotImplementedError):
        f(q, k, k, b, math.inf)
    with pytest.raises(ValueError):   # rows of the result that are not 16-byte addressable
        f(q, k, k, b, out=torch.empty(2, 4, 100, 68, dtype=q.dtype, device=DEV)[..., :64])


@pytest.mark.parametrize("change,rc", [(dict(B=-1), -2), (dict(Hq=3), -2), (dict(Hk=0), -2), (dict(Lk=-1), -2), (dict(count=-1), -2), (dict(D=32), -6), (dict(Lq=2 ** 31), -2), (dict(sm_scale=math.nan), -6), (dict(Lq=0), 0), (dict(B=0), 0),
                                       (dict(blocks=None), -1), (dict(o=None), -4), (dict(o_sl=12), -4), (dict(q=nv.Src4(None, 8, 8, 8)), -4), (dict(k=nv.Src4(64, 8, 8, 2 ** 25)), -2), (dict(v=nv.Src4(64, 8, 8, -8)), -2)])
def test_refusals_of_the_library(change, rc):
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    s = nv.Src4(p, 64, 64, 64)
    a = nv.SparseAttentionArgs(**{**dict(q=s, k=s, v=s, o=p, o_sb=64, o_sh=64, o_sl=64, blocks=p, B=1, Hq=2, Hk=2, Lq=128, Lk=128, count=1, D=64, sm_scale=1.0), **change})
    assert nv.lib().flux_sparse_attention_bf16(ctypes.byref(a), None, 0, None) == rc
    assert nv.lib().flux_sparse_attention_bf16(None, None, 0, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_lists_cut_in_parts(D):
    """Few query blocks with long lists: parts without a key, with scores of -inf, and one workspace for two captured graphs."""
    g = seeded(15)
    q, k, v = inputs(g, 1, 2, 1, 70, 64 * 40, D)
    blocks = lists(g, 1, 2, 70, 64 * 40, 40)
    blocks[0, 0, 0, 8:] = -1                      # the parts behind the first ones name nothing
    blocks[0, 1, 0, :32] = -1                     # ... in front of the last ones
    want = tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV))
    a = nv.SparseAttentionArgs(B=1, Hq=2, Hk=1, Lq=70, Lk=64 * 40, count=40, D=D)
    assert nv.lib().flux_sparse_attention_workspace_bytes(ctypes.byref(a)) > 0
    check(want, q, k, v, blocks)
    none = torch.full_like(blocks, -1)
    none[0, 1] = blocks[0, 1]
    got = tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), none.to(DEV))
    assert bool((got[0, 0] == 0).all()) and torch.equal(got[0, 1], want[0, 1])
    # keys whose scores are -inf beside others add nothing; where there are no others the formula is no number
    k2, q2 = k.clone(), q.clone()
    q2[..., 0] = q2[..., 0].abs() + 0.1
    first = int(blocks[0, 0, 0, 0])
    k2[0, 0, first * 64:first * 64 + 64, 0] = -math.inf
    some = blocks.clone()
    some[0, 1, 0, :], some[0, 1, 0, 3] = -1, first
    got = tk.block_sparse_attention(q2.to(DEV), k2.to(DEV), v.to(DEV), some.to(DEV)).cpu()
    rest = some.clone()
    rest[0, 0, 0, 0] = -1
    check(got[:, :1], q2[:, :1], k2, v, rest[:, :1])
    assert bool(got[0, 1].isnan().all())
    graphs, outs, args = [], [], [(q.to(DEV), blocks.to(DEV)), ((q * 2).to(DEV), some.to(DEV))]
    k, v = k.to(DEV), v.to(DEV)
    pool = None
    for qd, bd in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(tk.block_sparse_attention(qd, k, v, bd))
        pool = graph.pool()
        graphs.append(graph)
    for _ in range(3):
        for graph, out, (qd, bd) in zip(graphs, outs, args):
            graph.replay()
            assert torch.equal(out, tk.block_sparse_attention(qd, k, v, bd))
