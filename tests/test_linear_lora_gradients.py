"""linear_lora has no backward pass: a gradient that reaches it is an error, and calls whose gradients nobody asks for run as ever."""
import pytest
import torch

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded

BF = torch.bfloat16


class _Refuses:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_a_gradient_that_reaches_it_is_an_error(monkeypatch, native):
    if not native:
        monkeypatch.setattr(nv, "ops", lambda: _Refuses())
    g = seeded(1)
    operands = {"x": randn(g, 3, 20, 64, dtype=BF), "w": randn(g, 64, 64, dtype=BF, std=0.1), "b": randn(g, 64, dtype=BF), "lora_a": randn(g, 2, 8, 64, dtype=BF, std=0.1),
                "lora_b": randn(g, 2, 64, 8, dtype=BF), "scaling": torch.rand(2, generator=g)}
    operands = {k: t.to(DEV) for k, t in operands.items()}
    adapter = torch.tensor([1, -1, 0], device=DEV)
    plain = tk.linear_lora(**operands, adapter=adapter)
    assert not plain.requires_grad
    for name in operands:
        mine = {k: t.detach().requires_grad_(k == name) for k, t in operands.items()}
        y = tk.linear_lora(**mine, adapter=adapter)
        assert torch.equal(y, plain) and y.requires_grad
        assert torch.equal(y.detach(), plain)
        with pytest.raises(NotImplementedError, match="linear_lora is not differentiated"):
            y.float().sum().backward()
        with pytest.raises(NotImplementedError, match="linear_lora is not differentiated"):   # a branch beside it does not hide it
            (tk.layer_norm(mine["x"]) + y).float().sum().backward()
        assert mine[name].grad is None or name == "x"
        with torch.no_grad():
            assert not tk.linear_lora(**mine, adapter=adapter).requires_grad
        with torch.inference_mode():
            assert torch.equal(tk.linear_lora(**mine, adapter=adapter), plain)
    empty = tk.linear_lora(**{**operands, "x": operands["x"][:0].requires_grad_(True)}, adapter=adapter[:0])
    assert empty.shape == (0, 20, 64)


@pytest.mark.gpu
def test_forward_mode_and_transforms_are_refused():
    import torch.autograd.forward_ad as fwad

    g = seeded(2)
    x, w, a, b = randn(g, 3, 20, 64, dtype=BF).to(DEV), randn(g, 48, 64, dtype=BF).to(DEV), randn(g, 2, 8, 64, dtype=BF).to(DEV), randn(g, 2, 48, 8, dtype=BF).to(DEV)
    adapter = torch.tensor([1, -1, 0], device=DEV)
    for at in range(4):
        with fwad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            operands = [fwad.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate((x, w, a, b))]
            tk.linear_lora(operands[0], operands[1], None, *operands[2:], adapter)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: tk.linear_lora(t, w, None, a, b, adapter))(x[None])
