"""layer_norm of rows without values, and of no rows: results and gradients as torch.nn.functional.layer_norm has them."""
import pytest
import torch

import triton_kernels as tk
from util import DEV


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(0,), (3, 0), (2, 5, 0), (0, 0), (0, 7, 0), (0, 64), (2, 0, 64), (0, 4, 64)])
def test_no_values(shape, dtype):
    n = shape[-1]
    for w_shape in ((n,), None, (shape[0], *(1,) * (len(shape) - 2), n)):
        if w_shape is not None and len(shape) == 1 and w_shape != (n,):
            continue
        x = torch.empty(shape, device=DEV, dtype=dtype, requires_grad=True)
        w, b = (None if w_shape is None else torch.ones(w_shape, device=DEV, dtype=dtype, requires_grad=True) for _ in range(2))
        y = tk.layer_norm(x, w, b)
        assert y.shape == shape and y.dtype == dtype
        grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], torch.empty_like(y))
        assert grads[0].shape == shape
        for t in grads[1:]:
            assert t.shape == w_shape and t.dtype == dtype and (t == 0).all()
