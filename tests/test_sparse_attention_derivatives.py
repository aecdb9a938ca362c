"""Forward-mode derivatives of operands of block_sparse_attention whose result goes to `out`: an error, not nothing."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import triton_kernels as tk
from util import DEV, randn, seeded


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_tangents_of_a_call_with_a_given_result(device, at):
    g = seeded(at)
    q, k, v, out = (randn(g, 1, 2, 100, 64, dtype=torch.bfloat16).to(device) for _ in range(4))
    blocks, before = torch.zeros(1, 2, 1, 1, dtype=torch.int32, device=device), out.clone()
    with fwad.dual_level():
        operands = [fwad.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate((q, k, v, out))]
        with pytest.raises(NotImplementedError):
            tk.block_sparse_attention(*operands[:3], blocks, out=operands[3])
    assert torch.equal(out, before)


@pytest.mark.gpu
def test_within_a_level_without_tangents():
    g = seeded(9)
    q, k, v = (randn(g, 1, 2, 100, 64, dtype=torch.bfloat16).to(DEV) for _ in range(3))
    blocks, out = torch.zeros(1, 2, 1, 1, dtype=torch.int32, device=DEV), torch.empty_like(q)
    with fwad.dual_level():
        assert tk.block_sparse_attention(q, k, v, blocks, out=out) is out
    assert torch.equal(out, tk.block_sparse_attention(q, k, v, blocks))
