"""linear_lora: what is not finite in lora_b reaches its own rows as the formula has it, whoever else is in the batch."""
import pytest
import torch

import triton_kernels as tk
from util import DEV, randn, seeded

BF = torch.bfloat16


def make(seed, M, K, N, adapters, rank):
    g = seeded(seed)
    x, w = randn(g, M, K, dtype=BF).to(DEV), randn(g, N, K, dtype=BF, std=K ** -0.5).to(DEV)
    a, b = randn(g, adapters, rank, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, adapters, N, rank, dtype=BF, std=rank ** -0.5).to(DEV)
    return g, x, w, a, b, (0.5 + torch.rand(adapters, generator=g)).to(DEV)


def kinds(t):
    """0: finite, 1: +inf, 2: -inf, 3: NaN."""
    return t.isposinf() + 2 * t.isneginf() + 3 * t.isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 16, 24, 32, 40, 64])
@pytest.mark.parametrize("M,K,N", [(6, 512, 520), (40, 512, 520), (64, 16384, 2048), (700, 512, 1536), (2500, 256, 4096), (30, 100, 33)])
def test_what_is_not_finite_in_b_does_not_go_with_other_rows(M, K, N, rank):
    """Infinities and NaN come out as low * b has them, whoever else is in the batch: signs, both signs in one sum, zeros of low and infinite ones."""
    g, x, w, a, b, s = make(M + rank, M, K, N, 3, rank)
    inf, nan = float("inf"), float("nan")
    last, mid = rank - 1, rank // 2
    b[1, 3, 0], b[1, 4, last], b[1, 5, mid], b[1, N - 1, last] = inf, -inf, nan, -inf
    b[1, 8, 0], b[1, 8, last] = inf, -inf                       # (of one value where the rank is 1)
    b[1, 9, 0], b[1, 9, mid], b[1, 9, last] = -inf, -inf, -inf
    a[1, last, K // 2:], x[M - 1, : K // 2] = 0, 0               # low is zero there ...
    b[1, 12, 0] = 0
    x[2, 1] = inf                                               # ... and infinite or NaN here
    mixed = torch.randint(-1, 3, (M,), generator=g).to(DEV)
    mixed[2] = mixed[4] = mixed[M - 1] = 1
    alone = tk.linear_lora(x, w, None, a, b, torch.full_like(mixed, 1), s)
    got = tk.linear_lora(x, w, None, a, b, mixed, s)
    mine = mixed == 1
    assert torch.equal(kinds(got[mine]), kinds(alone[mine]))
    finite = alone.isfinite() & mine[:, None]
    assert torch.equal(got[finite], alone[finite])
    low = float(s[1]) * (x.double() @ a[1].double().T)
    low[M - 1, last] = 0.0
    want = kinds(x.double() @ w.double().T + (low[:, None, :] * b[1].double()).sum(-1)) if M * N * rank < 1 << 22 else None
    if want is not None:
        assert torch.equal(kinds(alone), want)
    others = mixed != 1
    clean = tk.linear_lora(x, w, None, a, torch.where(b.isfinite(), b, 0), mixed, s)
    assert torch.equal(got[others], clean[others])
    for row in (2, 4, M - 1):                                   # the row by itself, through the row-vector kernels
        assert torch.equal(kinds(tk.linear_lora(x[row:row + 1], w, None, a, b, mixed[row:row + 1], s)), kinds(got[row:row + 1]))
