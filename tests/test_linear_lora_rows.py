"""linear_lora of up to eight rows: weights of every size that the row-vector kernels take, in LDS and beside it, from one read to another."""
import pytest
import torch

import triton_kernels as tk
from test_linear_lora import check, make
from util import DEV


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("K,N", [(512, 64), (1536, 777), (3072, 23000), (6144, 12000), (12288, 300)])
def test_few_rows(M, K, N):
    g, x, w, b, lora_a, lora_b, scaling = make(M + K, (M,), K, N, 3, 40)
    adapter = torch.randint(-1, 3, (M,), generator=g).to(DEV)
    y = check(x, w, b, lora_a, lora_b, adapter, scaling)
    check(x, w, None, lora_a, lora_b, adapter, None, "GELU")
    assert torch.equal(tk.linear_lora(x, w, b, lora_a, lora_b, adapter, scaling), y)
