"""linear_lora's bias is one vector for all rows; anything else is refused (no GPU needed)."""
import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded

BF = torch.bfloat16


def operands():
    return torch.zeros(2, 3, 16, dtype=BF), torch.zeros(8, 16, dtype=BF), torch.zeros(4, 2, 16, dtype=BF), torch.zeros(4, 8, 2, dtype=BF), torch.zeros(2, dtype=torch.int32)


@pytest.mark.parametrize("shape", [(2, 8), (2, 1, 8), (3, 8), (0, 8), (7,), ()])
def test_other_shapes_are_refused(monkeypatch, shape):
    monkeypatch.setattr(nv, "require_gpu", lambda *t: t[0].device)
    x, w, a, b, i = operands()
    with pytest.raises(AssertionError, match="bias"):
        tk.linear_lora(x, w, torch.zeros(shape, dtype=BF), a, b, i)


@pytest.mark.gpu
def test_one_vector_in_any_shape():
    g = seeded(1)
    x, w, a, b, i = (t.to(DEV) for t in operands())
    bias = randn(g, 8, dtype=BF).to(DEV)
    want = tk.linear_lora(x, w, bias, a, b, i)
    assert torch.equal(want, bias.expand(2, 3, 8))
    for same in (bias[None], bias[None, None], torch.stack((bias, bias), 1)[:, 0], bias.float()):
        assert torch.equal(tk.linear_lora(x, w, same, a, b, i), want)
