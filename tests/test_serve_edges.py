"""Calls of linear_w4, select_blocks and block_sparse_attention at the edges of what they take."""
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
