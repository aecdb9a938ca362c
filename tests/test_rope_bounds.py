"""The bound that flux_hip_tune.h states for sines and cosines, against angles in 80 bits: 2^-23 beside |angle| (3 |log2 theta| + d / 5 + 5) 2^-53, d the values
of the axis. (The logarithm's 3 roundings and the power's own go with the exponent, at most |log2 theta|: ln 2 * 4 of it; three for every eighth pair; five besides.)"""
import numpy as np
import pytest
import torch

import triton_kernels as tk
from util import DEV


@pytest.mark.gpu
@pytest.mark.parametrize("theta", [10000.0, 1e6, 256.0, 0.01, 1.0, 3.7e11])
@pytest.mark.parametrize("axes", [(16, 56, 56), (512,), (2, 254), (64,)])
@pytest.mark.parametrize("far", [0, 10 ** 6, 2 ** 31 + 12345, 2 ** 36 + 1])
def test_tables_of_far_positions(far, axes, theta):
    if np.finfo(np.longdouble).nmant < 63:
        pytest.skip("no 80-bit numbers on this machine")
    L = 97
    ids = torch.stack([torch.arange(L, dtype=torch.int64) * (i + 1) + far for i in range(len(axes))], -1)
    wide = np.longdouble
    pos = ids.numpy().astype(wide)
    cols, bound = [], []
    for i, d in enumerate(axes):
        for j in range(d // 2):
            angle = pos[:, i] * np.power(wide(theta), wide(-2 * j) / wide(d))
            cols.append(angle)
            bound.append(2.0 ** -23 + np.abs(angle) * (3 * abs(np.log2(theta)) + d / 5 + 5) * 2.0 ** -53)
    angle, bound = np.stack(cols, -1), np.stack(bound, -1).astype(np.float64)
    want_c, want_s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    for at in (ids.to(DEV), ids.double().to(DEV), (-ids).to(DEV)):
        table = tk.rope_table(at, axes, theta)[0, 0].double().cpu().numpy()
        sign = -1.0 if at.flatten()[-1] < 0 else 1.0
        # (2^-60 of the angle: what 80 bits leave of it)
        off = bound + np.abs(angle).astype(np.float64) * 2.0 ** -60
        assert (np.abs(table[..., 0, 0] - want_c) <= off).all(), (np.abs(table[..., 0, 0] - want_c) - off).max()
        assert (np.abs(table[..., 1, 0] - sign * want_s) <= off).all(), (np.abs(table[..., 1, 0] - sign * want_s) - off).max()
