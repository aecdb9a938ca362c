"""Products with weights in 4 bits whose largest terms cancel, against float64 and the bound that the operator states: up to 128 rows a group's sum is that of
(q + 16) x less that of (z + 16) x."""
import pytest
import torch

import triton_kernels as tk
from util import DEV, seeded

HALF = torch.finfo(torch.bfloat16).eps / 2


def check(x, q, scale, zero, group, silu=False):
    z = 8.0 if zero is None else zero.double().repeat_interleave(group, 1)
    s = scale.double().repeat_interleave(group, 1)
    f = x.double() * torch.sigmoid(x.double()) if silu else x.double()
    want, size = f @ ((q.double() - z) * s).T, f.abs() @ ((32 + q.double() + z) * s).T
    # K + 8 sums and products, each good to 2^-23 of at most the sum of all terms' sizes (a product on the matrix cores may cut where it does not round);
    # x * sigmoid(x) is held to half a step of half a step, its exponential and reciprocal are good to 2^-20
    off = (x.shape[1] + 8) * 2.0 ** -23 * size + ((f.abs() @ ((q.double() - z).abs() * s).T) * (HALF ** 2 + 2.0 ** -19) if silu else 0)
    if x.shape[0] > 128:   # weights rounded to bf16: these are not, five bits times a scale of one
        assert torch.equal(((q.double() - z) * s).bfloat16().double(), (q.double() - z) * s)
    w = tk.pack_w4(q.to(DEV), scale.to(DEV), None if zero is None else zero.to(DEV))
    got = tk.linear_w4(x.to(DEV), w, in_activation="SiLU" if silu else "").double().cpu()
    assert bool(((got - want).abs() <= off + HALF * (want.abs() + off)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,silu", [(1, False), (1, True), (3, False), (8, True), (9, False), (24, False), (70, False), (128, False), (140, False)])
@pytest.mark.parametrize("small", [2.0 ** -17, 1.1875 * 2.0 ** -15, 2.0 ** -6])
def test_one_small_term_beside_many_that_are_nothing(rows, silu, small):
    """127 of a group's 128 columns have x = 1 and q = z = 15, one has q = 0 and is small."""
    q, scale, zero = torch.full((40, 256), 15), torch.full((40, 2), 0.5, dtype=torch.bfloat16), torch.full((40, 2), 15)
    x = torch.ones(rows, 256, dtype=torch.bfloat16)
    for n in range(40):
        q[n, (7 * n) % 256] = 0
    x[:, ::5] = small
    check(x, q, scale, zero, 128, silu)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 16, 40, 128, 200])
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 14, 2.0 ** 30])
@pytest.mark.parametrize("zeros", [False, True])
def test_outliers_that_meet_a_weight_of_nothing(rows, size, zeros):
    """A few columns of x are large, and their weights are 0 in half of the outputs."""
    g = seeded(rows)
    q, scale = torch.randint(0, 16, (48, 320), generator=g), torch.full((48, 5), 2.0 ** -4, dtype=torch.bfloat16)
    zero = torch.randint(0, 16, (48, 5), generator=g) if zeros else None
    x = torch.randn(rows, 320, generator=g).bfloat16()
    for k in (3, 64, 200, 319):
        x[:, k] *= size
        q[::2, k] = 8 if zero is None else zero[::2, k // 64]
    check(x, q, scale, zero, 64)
