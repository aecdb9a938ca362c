"""Weights in 4 bits at the edges of what they may be."""
import pytest
import torch

import triton_kernels as tk
from util import DEV, randn, seeded

BF = torch.bfloat16


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32, torch.uint64])
def test_numbers_of_every_whole_type(dtype, device):
    g = seeded(1)
    q, zero, scale = torch.randint(0, 16, (20, 96), generator=g), torch.randint(0, 16, (20, 3), generator=g), torch.rand(20, 3, generator=g).to(BF)
    q, zero, scale = q.to(device), zero.to(device), scale.to(device)
    w = tk.pack_w4(q.to(dtype), scale, zero.to(dtype))
    want = tk.pack_w4(q, scale, zero)
    assert torch.equal(w.packed, want.packed) and torch.equal(w.zero, want.zero) and torch.equal(w.scale, want.scale)
    for bad in ((q + 16).to(dtype), (q * 0 + 127).to(dtype)):
        with pytest.raises(ValueError):
            tk.pack_w4(bad, scale)
        with pytest.raises(ValueError):
            tk.pack_w4(q, scale, bad[:, :3])
    if dtype == torch.uint64:
        with pytest.raises(ValueError):
            tk.pack_w4(torch.full((20, 96), 2 ** 64 - 1, dtype=dtype).to(device), scale)


@pytest.mark.parametrize("zeros", [False, True])
def test_no_outputs(zeros):
    w = tk.quantize_w4(torch.zeros(0, 96), 32, zeros)
    assert w.shape == (0, 96) and w.packed.shape == (0, 1, 1024) and w.scale.shape == (0, 1, 16, 4)
    q, scale, zero = w.unpack()
    assert q.shape == (0, 96) and scale.shape == (0, 3) and (zero.shape == (0, 3) if zeros else zero is None)
    again = tk.pack_w4(q, scale, zero)
    assert again.shape == w.shape and again.packed.shape == w.packed.shape


@pytest.mark.gpu
def test_products_without_outputs():
    w = tk.quantize_w4(torch.zeros(0, 96, device=DEV), 32)
    for rows in (0, 1, 40, 200):
        assert tk.linear_w4(torch.zeros(rows, 96, dtype=BF, device=DEV), w).shape == (rows, 0)
    assert w.dequantize().shape == (0, 96)


def test_a_module_on_the_meta_device():
    """As other modules: made without memory, filled from a state dict."""
    from triton_kernels.modules import LinearW4

    lin = LinearW4(96, 40, group=32, zero_points=True, device="meta")
    assert lin.packed.is_meta and lin.weight.shape == (40, 96)
    from_weight = LinearW4.from_linear(torch.nn.Linear(96, 40), 32, True)
    lin.load_state_dict(from_weight.state_dict(), assign=True)
    assert all(torch.equal(a, b) for a, b in zip(lin.weight.unpack(), from_weight.weight.unpack())) and not lin.bias.requires_grad
    # one that is not filled is a weight of zeros
    q, scale, zero = LinearW4(96, 40, group=32).weight.unpack()
    assert zero is None and bool((scale == 0).all()) and q.shape == (40, 96)
