"""What the layer norm's backward pass asks of its workspace does not go with strides that nothing reads (no GPU needed)."""
import ctypes

import pytest

from triton_kernels import _native as nv

AT = 1 << 20   # an address, never read


def bytes_of(batch, seq, n, groups=1, dtype=0, **kw):
    a = nv.LayerNormBwdArgs(**{**dict(dy=AT, x=AT, w=AT, mean=AT, rstd=AT, dx=AT, dw=AT, db=AT, batch=batch, seq=seq, dy_sb=seq * n, dy_sl=n, x_sb=seq * n, x_sl=n,
                                      groups=groups, w_sb=n, n=n, x_dtype=dtype, w_dtype=dtype), **kw})
    return nv.lib().flux_layer_norm_bwd_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("dtype,widths", [(0, (768, 8200, 16384, 16392, 65536)), (1, (768, 8196, 12288, 12292, 65536))])
@pytest.mark.parametrize("batch", [129, 4096, 100000])
def test_one_row_a_batch_element(batch, dtype, widths):
    """[batch, 1, n] under one weight is [batch, n]: the stride of the dimension of one element is any number, and size and launch plan for the same rows."""
    for n in widths:
        want = bytes_of(1, batch, n, dtype=dtype)
        for odd in (0, 1, n + 1, -3, 1 << 40):
            assert bytes_of(batch, 1, n, dtype=dtype, dy_sl=odd) == bytes_of(batch, 1, n, dtype=dtype, x_sl=odd) == bytes_of(batch, 1, n, dtype=dtype, dy_sl=odd, x_sl=odd) == want
        # rows that are no 16-byte vectors are so in either form
        assert bytes_of(batch, 1, n, dtype=dtype, x_sb=n + 1) == bytes_of(1, batch, n, dtype=dtype, x_sl=n + 1)


@pytest.mark.parametrize("n", [768, 16384])
def test_other_dimensions_of_one_element(n):
    for odd in (0, 1, n + 1):
        assert bytes_of(1, 4096, n, dy_sb=odd, x_sb=odd) == bytes_of(1, 4096, n)
        assert bytes_of(1, 4096, n, w_sb=odd) == bytes_of(7, 4096, n, w_sb=odd, dy_sb=4096 * n, x_sb=4096 * n) == bytes_of(1, 4096, n)
        assert bytes_of(300, 1, n, groups=300, dy_sl=odd, x_sl=odd) == bytes_of(300, 1, n, groups=300)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,n", [(129, 16384), (300, 8200), (40, 768)])
def test_the_launch_stays_in_its_workspace(batch, n):
    """Through the C entry points with odd strides of the one-element dimension: the operator's own gradients, and what lies behind the workspace is left as it was."""
    import torch

    import triton_kernels as tk
    from util import DEV, randn, seeded

    g = seeded(n)
    x, dy = (randn(g, batch, n, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    w, b = (randn(g, n, dtype=torch.bfloat16).to(DEV).requires_grad_(True) for _ in range(2))
    leaf = x.clone().requires_grad_(True)
    want = torch.autograd.grad(tk.layer_norm(leaf, w, b), (leaf, w, b), dy)
    y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    stats = torch.empty(2, batch, device=DEV)
    lib, stream = nv.lib(), nv.stream_ptr(x.device)
    f = nv.LayerNormFwdArgs(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), batch, 1, n, n + 1, 1, 3, 5, n, 0, 0, 0, 1e-5)
    assert lib.flux_layer_norm(ctypes.byref(f), stream) == 0
    a = nv.LayerNormBwdArgs(dy.data_ptr(), x.data_ptr(), w.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), batch, 1, n, n + 1, n, 7, 1, 3, n, 0, 0, 0)
    need = lib.flux_layer_norm_bwd_workspace_bytes(ctypes.byref(a))
    room = torch.full((need + (64 << 20),), 0x5A, dtype=torch.uint8, device=DEV)
    assert lib.flux_layer_norm_bwd(ctypes.byref(a), room.data_ptr(), need, stream) == 0
    assert (room[need:] == 0x5A).all()
    for got, ref in zip((y, dx, dw, db), (tk.layer_norm(x, w, b).detach(), *want)):
        assert torch.equal(got, ref)
