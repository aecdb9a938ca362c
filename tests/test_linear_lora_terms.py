"""linear_lora's adapter terms by themselves: what is held between its two launches.

Tolerances. u = 2^-24. A sum of K products in fp32 is off by at most K u of the sum of their magnitudes. s x a^T is held as a bf16 number and what that
leaves over as another: 2^-8 of 2^-8 of its value. The result is rounded to bf16 once, 2^-8."""
import ctypes

import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded

BF, U = torch.bfloat16, 2.0 ** -24
# row vectors; eight-wave tiles with K whole and in parts; large tiles, with rows left over; no 16-byte rows
SHAPES = [(1, 64, 40), (3, 1024, 640), (8, 200, 4096), (7, 8192, 1000), (33, 512, 512), (64, 16384, 2048), (517, 2048, 2048), (2304, 1024, 3001), (4096, 512, 4096), (6000, 200, 3001), (12, 63, 50), (70, 1001, 65)]


def make(seed, M, K, N, adapters, rank):
    g = seeded(seed)
    x, w = randn(g, M, K, dtype=BF).to(DEV), randn(g, N, K, dtype=BF, std=K ** -0.5).to(DEV)
    a, b = randn(g, adapters, rank, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, adapters, N, rank, dtype=BF, std=rank ** -0.5).to(DEV)
    return g, x, w, a, b, (0.5 + torch.rand(adapters, generator=g)).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 16, 17, 40, 64, 250])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_terms_that_cancel_the_base_product(M, K, N, rank):
    """The bias takes out most of a row's result, so that the error of the adapter's terms is not hidden by the result's own rounding."""
    g, x, w, a, b, s = make(M + K + rank, M, K, N, 3, rank)
    owner = torch.randint(-1, 3, (M,), generator=g).sort().values.to(DEV)
    y, off, low = x.double() @ w.double().T, K * U * (x.double().abs() @ w.double().abs().T), torch.zeros(M, N, dtype=torch.float64, device=DEV)
    for i in range(3):
        at = (owner == i).nonzero()[:, 0]
        p = float(s[i]) * (x[at].double() @ a[i].double().T)
        low[at] = p @ b[i].double().T
        p_off = 2.0 ** -16 * p.abs() + 2 * K * U * float(s[i]) * (x[at].double().abs() @ a[i].double().abs().T)
        off[at] += p_off @ b[i].double().abs().T + 2 * rank * U * (p.abs() @ b[i].double().abs().T)
    bias = (-(y + low)[M // 2]).to(BF)
    want = y + low + bias.double()
    off += 4 * U * (y.abs() + low.abs() + bias.double().abs())
    err = (tk.linear_lora(x, w, bias, a, b, owner, s).double() - want).abs()
    assert (err <= off + 2.0 ** -8 * want.abs()).all(), (err - off - 2.0 ** -8 * want.abs()).max()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,rank,once", [(300, 256, 520, 64, True), (2304, 512, 1536, 100, True), (9, 256, 64, 17, True), (64, 128, 96, 16, False), (5, 512, 384, 40, False), (20, 63, 50, 33, False)])
def test_what_the_workspace_has_room_for(M, K, N, rank, once):
    """In tiles and beyond rank 16 the least workspace holds one number a term, 2^-8 of it off; twice that holds what linear_lora itself computes with."""
    g, x, w, a, b, s = make(M + rank, M, K, N, 3, rank)
    owner = torch.randint(-1, 3, (M,), generator=g, dtype=torch.int32).sort().values.to(DEV)
    want, lib = tk.linear_lora(x, w, None, a, b, owner, s), nv.lib()
    outs = []
    for times in (1, 2):
        y = torch.empty_like(want)
        args = nv.LinearLoraArgs(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), a.data_ptr(), b.data_ptr(), owner.data_ptr(), s.data_ptr(), M, N, K, K, K, N, M, 3, rank, 0, 0)
        room = times * lib.flux_linear_lora_least_bytes(ctypes.byref(args))
        ws = torch.full((room + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
        assert lib.flux_linear_lora_bf16(ctypes.byref(args), ws.data_ptr(), room, nv.stream_ptr(x.device)) == 0
        assert (ws[room:] == 0x5A).all()
        outs.append(y)
    assert torch.equal(outs[1], want) and torch.equal(outs[0], want) != once
    low = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    off = torch.zeros_like(low)
    for i in range(3):
        at = (owner == i).nonzero()[:, 0]
        p = float(s[i]) * (x[at].double() @ a[i].double().T)
        low[at], off[at] = p @ b[i].double().T, (2.0 ** -8 * p.abs() + 2 * K * U * float(s[i]) * (x[at].double().abs() @ a[i].double().abs().T)) @ b[i].double().abs().T
    exact = x.double() @ w.double().T + low
    off += (K + rank + 4) * U * (x.double().abs() @ w.double().abs().T + low.abs()) + rank * U * off * 2 ** 8
    assert ((outs[0].double() - exact).abs() <= off + 2.0 ** -8 * exact.abs()).all()
