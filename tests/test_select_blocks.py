"""Which blocks of keys the blocks of queries attend to, against means, products and an order formed in float64 on the CPU, and what is refused."""
import ctypes
import math

import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded


def expected(q, k, keep, always=0, lengths=None):
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    count = -(-Lk // 64)
    out = torch.full((B, Hq, -(-Lq // 128), min(keep, count)), -1, dtype=torch.int32)
    for b in range(B):
        end = Lk if lengths is None else min(max(int(lengths[b]), 0), Lk)
        have = -(-end // 64)
        for h in range(Hq):
            if have == 0:
                continue
            mq = torch.stack([t.double().mean(0) for t in q[b, h].split(128)])
            mk = torch.stack([t.double().mean(0) for t in k[b, h // (Hq // Hk), :end].split(64)])
            for t, m in enumerate(mq):
                score = [math.inf if j < always else float((m * row).sum()) for j, row in enumerate(mk)]
                # (a NaN behind everything, the first blocks in front of everything)
                order = sorted(range(have), key=lambda j: (j >= always, math.isnan(score[j]), 0.0 if math.isnan(score[j]) else -score[j], j))
                chosen = sorted(order[:keep])
                out[b, h, t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out


def inputs(g, B, Hq, Hk, Lq, Lk, D):
    return randn(g, B, Lq, Hq, D, dtype=torch.bfloat16).transpose(1, 2), randn(g, B, Lk, Hk, D, dtype=torch.bfloat16).transpose(1, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hq,Hk,Lq,Lk,D,keep,always,padded", [
    (1, 1, 1, 1, 1, 64, 1, 0, False), (1, 2, 1, 128, 64, 128, 1, 0, False), (2, 4, 2, 129, 65, 64, 1, 0, True), (1, 3, 3, 640, 640, 128, 3, 0, False), (2, 2, 2, 1084, 1084, 64, 5, 1, True),
    (3, 4, 1, 1, 2000, 128, 7, 2, True), (1, 2, 2, 2300, 4608, 128, 18, 8, False), (1, 1, 1, 257, 16384, 64, 100, 0, False), (1, 1, 1, 200, 16450, 128, 1, 0, False), (2, 1, 1, 130, 33000, 64, 64, 3, True),
    (1, 2, 1, 300, 66000, 64, 40, 0, False), (1, 1, 1, 4000, 700, 128, 50, 0, False), (1, 8, 8, 17, 1000, 64, 16, 20, False), (1, 1, 1, 2100, 320, 64, 4, 0, False)])
def test_against_float64(B, Hq, Hk, Lq, Lk, D, keep, always, padded):
    g = seeded(Lq + Lk)
    q, k = inputs(g, B, Hq, Hk, Lq, Lk, D)
    lengths = torch.tensor([Lk, max(Lk // 3, 1), 0][:B], dtype=torch.int32) if padded else None
    got = tk.select_blocks(q.to(DEV), k.to(DEV), keep, always=always, lengths=None if lengths is None else lengths.to(DEV))
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), expected(q, k, keep, always, lengths))


@pytest.mark.gpu
def test_the_lower_number_goes_first_among_equals():
    g = seeded(2)
    q, k = inputs(g, 1, 2, 2, 260, 64 * 90, 128)
    k[:] = k[:, :, :64].repeat(1, 1, 90, 1)                     # all alike
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 7).cpu(), torch.arange(7, dtype=torch.int32).expand(1, 2, 3, 7))
    k[:, :, 64 * 80:64 * 83] = k[:, :, 64 * 80:64 * 83] * 2     # three others, alike, above or beneath
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 5).cpu(), expected(q, k, 5))
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 2).cpu(), expected(q, k, 2))
    zero = torch.zeros_like(k)
    zero[:, :, ::2] = -0.0                                      # 0 and -0 are equals
    assert torch.equal(tk.select_blocks(q.to(DEV), zero.to(DEV), 4).cpu(), torch.arange(4, dtype=torch.int32).expand(1, 2, 3, 4))


@pytest.mark.gpu
def test_values_that_are_not_finite():
    g = seeded(3)
    q, k = inputs(g, 1, 1, 1, 256, 640, 64)
    k[0, 0, 70], k[0, 0, 200, 3], k[0, 0, 330, 5] = math.nan, math.inf, -math.inf
    q[0, 0, :128, 3], q[0, 0, :128, 5] = q[0, 0, :128, 3].abs(), q[0, 0, :128, 5].abs()
    for keep in (1, 4, 9, 10):
        assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), keep).cpu(), expected(q, k, keep))
    q[0, 0, 130] = math.nan
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 3).cpu()[0, 0, 1], torch.arange(3, dtype=torch.int32))


@pytest.mark.gpu
def test_keys_behind_the_length_are_not_looked_at():
    g = seeded(4)
    q, k = inputs(g, 3, 2, 1, 150, 400, 128)
    lengths = torch.tensor([100, 0, 257])
    want = expected(q, k, 4, 1, lengths)
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n:] = math.nan
    for kind in (torch.int32, torch.int64, torch.int16):
        assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 4, always=1, lengths=lengths.to(DEV, kind)).cpu(), want)
    k[:] = torch.nan_to_num(k)
    far = torch.tensor([2 ** 33, -5, 401], device=DEV)          # beyond the end, below 0
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 4, lengths=far).cpu(), expected(q, k, 4, 0, far.tolist()))
    assert bool((tk.select_blocks(q.to(DEV), k.to(DEV), 4, lengths=far)[1] == -1).all())


@pytest.mark.gpu
def test_views_streams_graphs_and_nothing():
    g = seeded(5)
    wide = randn(g, 2, 500, 3, 4, 136, dtype=torch.bfloat16).to(DEV)
    q, k = wide[:, :, 0, :, :128].transpose(1, 2), wide[:, 20:, 1, :2, 8:].transpose(1, 2)
    want = expected(q.cpu(), k.cpu(), 3)
    assert torch.equal(tk.select_blocks(q, k, 3).cpu(), want)
    odd = wide[:, :, 0, :, 1:129].transpose(1, 2)
    assert torch.equal(tk.select_blocks(odd, k, 3).cpu(), expected(odd.cpu(), k.cpu(), 3))
    assert tk.select_blocks(q, k, 0).shape == (2, 4, 4, 0) and tk.select_blocks(q[:, :, :0], k, 3).shape == (2, 4, 0, 3) and tk.select_blocks(q, k[:, :, :0], 3).shape == (2, 4, 4, 0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(tk.select_blocks(q, k, 3).cpu(), want)
    mine, graph = q.clone(), torch.cuda.CUDAGraph()
    tk.select_blocks(mine, k, 3)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = tk.select_blocks(mine, k, 3)
    for i in range(3):
        mine.copy_(randn(g, 2, 4, 500, 128, dtype=torch.bfloat16))
        graph.replay()
        assert torch.equal(out, tk.select_blocks(mine, k, 3))
    assert not tk.select_blocks(q.clone().requires_grad_(True), k, 3).requires_grad


@pytest.mark.gpu
def test_refusals_of_a_call():
    q, k = torch.zeros(2, 4, 100, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 2, 100, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: tk.select_blocks(q[0], k, 1), lambda: tk.select_blocks(q, k[:1], 1), lambda: tk.select_blocks(q[:, :3], k, 1), lambda: tk.select_blocks(q[..., :32], k[..., :32], 1), lambda: tk.select_blocks(q, k, -1),
                lambda: tk.select_blocks(q, k, 1, always=-1), lambda: tk.select_blocks(q, k, 1, lengths=torch.zeros(3, dtype=torch.int32, device=DEV))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        tk.select_blocks(q.float(), k.float(), 1)
    with pytest.raises(TypeError):
        tk.select_blocks(q, k, 1, lengths=torch.zeros(2, device=DEV))
    with pytest.raises(RuntimeError):
        tk.select_blocks(q, k.cpu(), 1)
    with pytest.raises(NotImplementedError):   # 16385 blocks of keys
        tk.select_blocks(q[:1, :1], k[:1, :1, :1].expand(1, 1, 64 * 16384 + 1, 64), 1)


@pytest.mark.parametrize("change,rc", [(dict(B=-1), -2), (dict(Hq=3), -2), (dict(Hk=0), -2), (dict(Lk=-1), -2), (dict(keep=-1), -2), (dict(always=-1), -2), (dict(D=32), -6), (dict(Lk=64 * 16384 + 1), -6), (dict(Lq=2 ** 31), -2),
                                       (dict(keep=0), 0), (dict(Lq=0), 0), (dict(blocks=None), -1), (dict(q=nv.Src4(None, 8, 8, 8)), -4), (dict(k=nv.Src4(64, 8, 8, 12)), -4), (dict(), -2)])
def test_refusals_of_the_library(change, rc):
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    a = nv.SelectBlocksArgs(**{**dict(q=nv.Src4(p, 64, 64, 64), k=nv.Src4(p, 64, 64, 64), blocks=p, B=1, Hq=2, Hk=2, Lq=128, Lk=128, keep=1, always=0, D=64), **change})
    need = nv.lib().flux_select_blocks_workspace_bytes(ctypes.byref(a))
    assert (need > 0) == (rc in (-1, -4) or not change)
    assert nv.lib().flux_select_blocks(ctypes.byref(a), p, need - 1 if not change else 1 << 30, None) == rc
    assert nv.lib().flux_select_blocks(None, None, 0, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("D,L", [(64, 64 * 100), (128, 64 * 300), (64, 64 * 700)])
@pytest.mark.parametrize("close", [2.0 ** -7, 2.0 ** -16, 0.0])
def test_scores_that_lie_close_together(D, L, close):
    """Blocks of keys that are nearly alike, of a few kinds: neighbours differ by one bf16 step of one value, or by a large common value that all share, or not at all."""
    g = seeded(D)
    q = randn(g, 1, 1, 140, D, dtype=torch.bfloat16)
    kinds = randn(g, 5, 64, D, dtype=torch.bfloat16)
    k = kinds[torch.randint(0, 5, (L // 64,), generator=g)].reshape(1, 1, L, D).clone()
    at = torch.arange(0, L, 64) + torch.randint(0, 64, (L // 64,), generator=g)
    column = torch.randint(0, D, (L // 64,), generator=g)
    k[0, 0, at, column] += (k[0, 0, at, column].float() * close * torch.randint(-3, 4, (L // 64,), generator=g)).to(torch.bfloat16)
    k[..., 0] += 200.0   # scores are the same to 2^-10 of them and more
    q[..., 0] += 50.0
    for keep in (1, 7, L // 64 // 3, L // 64 - 1):
        assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), keep, always=1).cpu(), expected(q, k, keep, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-19, 1e12, 1e30])
def test_scores_of_other_sizes(size):
    g = seeded(7)
    q, k = inputs(g, 1, 2, 1, 300, 64 * 150, 128)
    q, k = (q.float() * size).bfloat16(), (k.float() * size).bfloat16()
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 20).cpu(), expected(q, k, 20))
    k[:, :, ::3] = (k[:, :, ::3].float() / max(size, 1e-20) * 1e-3).bfloat16()   # among others of ordinary size
    assert torch.equal(tk.select_blocks(q.to(DEV), k.to(DEV), 20).cpu(), expected(q, k, 20))
