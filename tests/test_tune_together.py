"""layer_norm, linear_lora, apply_rope_nd and rope_table as a block uses them: one block served to requests with adapters of their own, and one
training step through the normalisation and the rotation."""
import math

import pytest
import torch

import triton_kernels as tk
from triton_kernels import testing as cfg
from util import DEV, randn, seeded

BF, U = torch.bfloat16, 2.0 ** -24
AXES = [16, 56, 56]


def lora64(x, w, b, lora_a, lora_b, adapter, scaling, gelu=False):
    """The projection in 64 bits and the bound that its own test derives."""
    import test_linear_lora
    return test_linear_lora.exact(x, w, b, lora_a, lora_b, adapter, scaling, gelu)


@pytest.mark.gpu
@pytest.mark.parametrize("B,text,grid", [(3, 17, 16), (1, 5, 4), (2, 100, 64)])
def test_one_block_for_many_requests(B, text, grid):
    """adaLN, the q, k and v projection with an adapter a request, q/k norm, rotation by three axes, attention, projection and GELU with adapters. Every
    operator is held against 64 bits on what the run before it gave it; the run gives the same bits again and out of a graph."""
    H, D = 4, 128
    K = H * D
    g = seeded(B + text)
    L = text + (grid // 2) ** 2
    x, mod = randn(g, B, L, K, dtype=BF).to(DEV), randn(g, B, 1, 2 * K, dtype=BF, std=0.2).to(DEV)
    w_qkv, b_qkv, w_up = randn(g, 3 * K, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, 3 * K, dtype=BF, std=0.1).to(DEV), randn(g, 4 * K, K, dtype=BF, std=K ** -0.5).to(DEV)
    a_qkv, b_lora = randn(g, 5, 12, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, 5, 3 * K, 12, dtype=BF, std=0.3).to(DEV)
    a_up, b_up, scaling = randn(g, 5, 40, K, dtype=BF, std=K ** -0.5).to(DEV), randn(g, 5, 4 * K, 40, dtype=BF, std=0.2).to(DEV), torch.rand(5, generator=g).to(DEV)
    adapter = torch.tensor([4, -1, 2][:B], dtype=torch.int32, device=DEV)
    q_scale, k_scale = (1 + 0.1 * randn(g, D)).to(DEV), (1 + 0.1 * randn(g, D)).to(DEV)
    ids = cfg.flux_position_ids(text, grid // 2).to(DEV)
    assert ids.shape[-2] == L

    def run():
        h = tk.layer_norm(x, mod[..., :K], mod[..., K:], 1e-6, plus_one=True)
        qkv = tk.linear_lora(h, w_qkv, b_qkv, a_qkv, b_lora, adapter, scaling)
        q, k, v = qkv.view(B, L, 3, H, D).permute(2, 0, 3, 1, 4)
        qn, kn = tk.rms_norm(q, q_scale, 1e-6), tk.rms_norm(k, k_scale, 1e-6)
        qr, kr = tk.apply_rope_nd(qn, kn, ids, AXES)
        o = tk.scaled_dot_product_attention(qr, kr, v)
        flat = o.transpose(1, 2).reshape(B, L, K)
        return h, qkv, qn, kn, qr, kr, flat, tk.linear_lora(flat, w_up, None, a_up, b_up, adapter, scaling, "GELU")

    with torch.no_grad():
        h, qkv, qn, kn, qr, kr, o, up = run()
    xd = x.double()
    var, mean = torch.var_mean(xd, -1, correction=0, keepdim=True)
    n = (xd - mean) / torch.sqrt(var + 1e-6)
    want = n * (1 + mod[..., :K].double()) + mod[..., K:].double()
    off = 512 * U * (1 + n.abs()) * (1 + mod[..., :K].double()).abs() + 4 * U * (want.abs() + n.abs() * 2 + 1)
    assert ((h.double() - want).abs() <= off + 2.0 ** -8 * want.abs()).all()
    for got, (y, y_off) in ((qkv, lora64(h, w_qkv, b_qkv, a_qkv, b_lora, adapter, scaling)), (up, lora64(o, w_up, None, a_up, b_up, adapter, scaling, True))):
        assert ((got.double() - y).abs() <= y_off + 2.0 ** -8 * y.abs()).all()
    # rotation: with the 64-bit table and with rope_table's through apply_rope
    angle = torch.cat([ids[..., i].double()[..., None] / 10000.0 ** (2 * torch.arange(d // 2, device=DEV).double() / d) for i, d in enumerate(AXES)], -1).view(1, 1, L, -1)
    for src, got in ((qn, qr), (kn, kr)):
        s = src.double().unflatten(-1, (-1, 2))
        t = torch.stack((s[..., 0] * angle.cos() - s[..., 1] * angle.sin(), s[..., 0] * angle.sin() + s[..., 1] * angle.cos()), -1).flatten(-2)
        size = s.abs().sum(-1).repeat_interleave(2, -1)
        assert ((got.double() - t).abs() <= 2.0 ** -21 * size + 2.0 ** -8 * t.abs()).all()
    table = tk.EmbedND(128, 10000, AXES)(ids)
    for one, two in zip(tk.apply_rope(qn, kn, table), (qr, kr)):     # (one more rounding of each product's factors there)
        assert ((one.double() - two.double()).abs() <= 2.0 ** -7 * two.double().abs() + 2.0 ** -20 * qn.abs().max().double()).all()
    # the adapters matter, each to its own request alone
    none = tk.linear(h, w_qkv, b_qkv)
    for i, own in enumerate(adapter.tolist()):
        assert torch.equal(none[i], qkv[i]) == (own < 0)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(run(), (h, qkv, qn, kn, qr, kr, o, up)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        for i in range(3):
            x.copy_(randn(g, B, L, K, dtype=BF))
            adapter.copy_(torch.randint(-1, 5, (B,), generator=g, dtype=torch.int32))
            ids.add_(1)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(held, run()))
            torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("B,frames,height,width,each", [(2, 3, 4, 5, True), (1, 2, 7, 9, False), (3, 1, 1, 2, True)])
def test_a_training_step_through_both(B, frames, height, width, each):
    """Gradients of adaLN's scale and shift, of a trained projection and of x through attention over rotated q and k, in fp32 beside the same step in
    64 bits. A sum of n products carries n / 2 u of its magnitudes on average over fewer than 2^10 of them, here through five products and a softmax
    whose scores stay below 16 in size: 2^-24 * 2^10 * 6 * 16 < 2^-7 at the very worst and, with errors of either sign, 2^-24 * 2^5 * 6 * 16 < 2^-12."""
    H, D = 2, 64
    K, L, axes = H * D, frames * height * width, (16, 24, 24)
    g = seeded(L)
    ids = torch.cartesian_prod(torch.arange(frames), torch.arange(height), torch.arange(width)).to(DEV)
    x, w = randn(g, B, L, K).to(DEV), randn(g, 3 * K, K, std=K ** -0.5).to(DEV)
    scale, shift = (randn(g, *((B, 1, K) if each else (K,)), std=0.3).to(DEV) for _ in range(2))
    dy = randn(g, B, L, K).to(DEV)

    def step(x, w, scale, shift, norm, rope):
        h = norm(x, scale, shift)
        q, k, v = (h @ w.T).view(B, L, 3, H, D).permute(2, 0, 3, 1, 4)
        q, k = rope(q, k)
        p = torch.softmax((q.unsqueeze(3) * k.unsqueeze(2)).sum(-1) / math.sqrt(D), -1)
        return (p.unsqueeze(-1) * v.unsqueeze(2)).sum(3).transpose(1, 2).reshape(B, L, K)

    leaves = [t.clone().requires_grad_(True) for t in (x, w, scale, shift)]
    y = step(*leaves, lambda x, s, b: tk.layer_norm(x, s, b, 1e-6, plus_one=True), lambda q, k: tk.apply_rope_nd(q, k, ids, axes))
    grads = torch.autograd.grad(y, leaves, dy)

    angle = torch.cat([ids[:, i].double()[:, None] / 10000.0 ** (2 * torch.arange(d // 2, device=DEV).double() / d) for i, d in enumerate(axes)], -1)

    def turn(t):
        t = t.unflatten(-1, (-1, 2))
        return torch.stack((t[..., 0] * angle.cos() - t[..., 1] * angle.sin(), t[..., 0] * angle.sin() + t[..., 1] * angle.cos()), -1).flatten(-2)

    exact = [t.double().requires_grad_(True) for t in (x, w, scale, shift)]
    want = step(*exact, lambda x, s, b: torch.nn.functional.layer_norm(x, (K,), eps=1e-6) * (1 + s) + b, lambda q, k: (turn(q), turn(k)))
    for got, ref in zip((y, *grads), (want, *torch.autograd.grad(want, exact, dy.double()))):
        assert got.shape == ref.shape and (got.double() - ref).norm() <= 2.0 ** -12 * ref.norm()


@pytest.mark.gpu
def test_a_captured_training_step():
    """Forward and backward in one graph, replayed between eager steps over other leaves."""
    g = seeded(7)
    B, L, H, D, axes = 2, 40, 3, 64, (16, 24, 24)
    ids = torch.randint(0, 30, (B, L, 3), generator=g).to(DEV)
    held = [randn(g, B, L, H * D, dtype=BF).to(DEV), randn(g, H * D, dtype=BF).to(DEV), randn(g, H * D, dtype=BF).to(DEV), randn(g, B, H, L, D, dtype=BF).to(DEV)]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in held[:3]]
        heads = tk.layer_norm(*leaves).view(B, L, H, D).transpose(1, 2)
        q, k = tk.apply_rope_nd(heads, heads[:, :1], ids, axes)
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (held[3], held[3][:, :1]))]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        for t in held:
            t.copy_(randn(g, *t.shape, dtype=BF))
        ids.add_(2)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
        torch.cuda.synchronize()
