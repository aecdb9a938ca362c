"""linear_w4, select_blocks and block_sparse_attention in native code (csrc/torch_ops.cpp) against the Python launchers of the same operators: the same bits, and the
calls that are left to the launchers."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwad

import triton_kernels as tk
from triton_kernels import _native as nv
from test_tune_native_calls import launcher, took
from util import DEV, randn, seeded

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def weight(g, n=48, k=192, zeros=True):
    q = torch.randint(0, 16, (n, k), generator=g)
    return tk.pack_w4(q.to(DEV), torch.rand(n, k // 64, generator=g).to(DEV, BF), torch.randint(0, 16, (n, k // 64), generator=g).to(DEV) if zeros else None)


def sparse(g, B=2, Hq=4, Hk=2, L=300, D=64):
    q = randn(g, B, L, Hq, D, dtype=BF).to(DEV).transpose(1, 2)
    k, v = (randn(g, B, L, Hk, D, dtype=BF).to(DEV).transpose(1, 2) for _ in range(2))
    return q, k, v, torch.randint(-1, 6, (B, Hq, -(-L // 128), 3), generator=g, dtype=torch.int32).to(DEV)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows", [1, 6, 20, 140])
def test_linear_w4(monkeypatch, zeros, rows):
    g = seeded(rows)
    w = weight(g, zeros=zeros)
    x, b = randn(g, rows, 2 * 192, dtype=BF).to(DEV)[:, :192], randn(g, 48, dtype=BF).to(DEV)
    for args, kw in (((x, w, b), {}), ((x, w), dict(activation="GELU")), ((x[None], w, b), {}), ((x[0], w, b), dict(in_activation="SiLU"))):
        assert took(monkeypatch, tk.linear_w4, *args, **kw)
        a, c = tk.linear_w4(*args, **kw), launcher(monkeypatch, tk.linear_w4, *args, **kw)
        assert a.shape == c.shape and a.stride() == c.stride() and torch.equal(a, c)


def test_linear_w4_left_to_the_launcher(monkeypatch):
    g = seeded(1)
    w, x = weight(g), randn(g, 4, 400, dtype=BF).to(DEV)
    for args, kw in (((x[:, 3:195], w), {}), ((x[:, :384:2], w), {}), ((x[:0, :192], w), {}), ((x[:, :192], w, torch.zeros(48, device=DEV)), {}), ((x[:, :192].clone().requires_grad_(True), w), {})):
        assert not took(monkeypatch, tk.linear_w4, *args, **kw)
    with torch.no_grad():
        assert took(monkeypatch, tk.linear_w4, x[:, :192].clone().requires_grad_(True), w)
    y = tk.linear_w4(x[:, :192].clone().requires_grad_(True), w)
    with pytest.raises(NotImplementedError):
        y.sum().backward()
    with fwad.dual_level(), pytest.raises(Exception):
        tk.linear_w4(fwad.make_dual(x[:, :192].clone(), torch.ones_like(x[:, :192])), w)
    with pytest.raises(NotImplementedError):
        tk.linear_w4(x[:, :192].repeat(3, 1), w, in_activation="SiLU")
    with pytest.raises(RuntimeError):
        tk.linear_w4(x[:, :192], w.to("cpu"))


def test_select_blocks(monkeypatch):
    q, k, _, _ = sparse(seeded(2))
    lengths = torch.tensor([300, 70], dtype=torch.int32, device=DEV)
    for args, kw in (((q, k, 2), {}), ((q, k, 9), dict(always=1)), ((q, k, 2), dict(lengths=lengths))):
        assert took(monkeypatch, tk.select_blocks, *args, **kw)
        assert torch.equal(tk.select_blocks(*args, **kw), launcher(monkeypatch, tk.select_blocks, *args, **kw))
    for args, kw in (((q, k, 0), {}), ((q[:, :, :0], k, 2), {}), ((q, k, 2), dict(lengths=lengths.long())), ((q, k, torch.tensor(2)), {})):
        assert not took(monkeypatch, tk.select_blocks, *args, **kw)
    assert torch.equal(tk.select_blocks(q, k, 2, lengths=lengths.long()), tk.select_blocks(q, k, 2, lengths=lengths))
    with pytest.raises(AssertionError):
        tk.select_blocks(q, k, 2, always=-1)


def test_block_sparse_attention(monkeypatch):
    q, k, v, blocks = sparse(seeded(3))
    lengths = torch.tensor([300, 70], dtype=torch.int32, device=DEV)
    out = torch.empty(2, 300, 4, 64, dtype=BF, device=DEV).transpose(1, 2)
    for args, kw in (((q, k, v, blocks), {}), ((q, k, v, blocks, 0.2), {}), ((q, k, v, blocks), dict(lengths=lengths)), ((q, k, v, blocks), dict(out=out))):
        assert took(monkeypatch, tk.block_sparse_attention, *args, **kw)
        a = tk.block_sparse_attention(*args, **kw).clone()
        assert torch.equal(a, launcher(monkeypatch, tk.block_sparse_attention, *args, **kw))
    for args, kw in (((q, k, v, blocks.long()), {}), ((q, k, v, blocks[..., :0]), {}), ((q, k, v, blocks.repeat_interleave(2, -1)[..., ::2]), {}), ((q, k, v, blocks), dict(lengths=lengths.long())),
                     ((q.clone().requires_grad_(True), k, v, blocks), {})):
        assert not took(monkeypatch, tk.block_sparse_attention, *args, **kw)
    with fwad.dual_level(), pytest.raises(Exception):
        tk.block_sparse_attention(fwad.make_dual(q.clone(), torch.ones_like(q)), k, v, blocks)
    with pytest.raises(NotImplementedError):
        tk.block_sparse_attention(q, k, v, blocks, float("nan"))


def test_calls_of_several_threads():
    g = seeded(4)
    w, x = weight(g), randn(g, 8, 192, dtype=BF).to(DEV)
    q, k, v, blocks = sparse(g)
    want = tk.linear_w4(x, w), tk.select_blocks(q, k, 2), tk.block_sparse_attention(q, k, v, blocks)
    torch.cuda.synchronize()
    wrong = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = tk.linear_w4(x, w), tk.select_blocks(q, k, 2), tk.block_sparse_attention(q, k, v, blocks)
                stream.synchronize()
                wrong.extend(i for i in range(3) if not torch.equal(got[i], want[i]))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
