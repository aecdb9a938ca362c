"""Blocks that serve with a modulation in 4 bits and attention over selected blocks: modules, state dicts, and the operators one behind the other as a block has them."""
import copy

import pytest
import torch
import torch.nn.functional as F

import triton_kernels as tk
from triton_kernels.modules import Linear, LinearW4, Modulation
from util import DEV, randn, seeded

BF = torch.bfloat16
HALF = torch.finfo(BF).eps / 2


def block(cls, hidden, heads, seed=0, **kw):
    torch.manual_seed(seed)
    return cls(hidden, heads, **kw).to(BF)


def test_linear_w4_module_on_the_cpu():
    lin = Linear(192, 40).to(BF)
    w4 = LinearW4.from_linear(lin, 64, True)
    want = tk.quantize_w4(lin.weight, 64, True)
    assert w4.weight.shape == (40, 192) and torch.equal(w4.packed, want.packed) and torch.equal(w4.scale, want.scale) and torch.equal(w4.zero, want.zero)
    assert torch.equal(w4.bias, lin.bias) and w4.bias.data_ptr() != lin.bias.data_ptr() and not any(p.requires_grad for p in w4.parameters())
    other = LinearW4(192, 40, group=64, zero_points=True)
    other.load_state_dict(w4.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(other.state_dict().values(), w4.state_dict().values()))
    assert LinearW4(192, 40, bias=False).bias is None and "zero" not in LinearW4(192, 40).state_dict()
    with pytest.raises(AssertionError):
        LinearW4(100, 40)
    with pytest.raises(AssertionError):
        w4.float().weight   # scales are bf16


@pytest.mark.gpu
@pytest.mark.parametrize("rows,double", [(1, True), (3, False), (12, False)])
def test_modulation_in_4_bits(rows, double):
    m = block(Modulation, 256, double)
    vec = randn(seeded(rows), rows, 256, dtype=BF)
    w4 = LinearW4.from_linear(m.lin, 64, True)
    q, scale, zero = w4.weight.unpack()
    # (beyond 8 rows SiLU is an operator of its own, rounded to bf16: half a step of every value)
    want = tk.linear_w4_torch(vec, q, scale, zero, m.lin.bias, in_activation="SiLU").double()
    m = m.to(DEV).quantize(64, True)
    assert isinstance(m.lin, LinearW4) and m.lin.packed.is_cuda
    first, second = m(vec.to(DEV))
    assert (second is not None) == double
    got = torch.cat([t for o in (first, second) if o is not None for t in (o.shift, o.scale, o.gate)], -1)[:, 0]
    w = ((q.double().unflatten(1, (-1, 64)) - zero.double()[..., None]) * scale.double()[..., None]).flatten(1)
    size = F.silu(vec.double()).abs() @ w.abs().T
    assert bool(((got.double().cpu() - want).abs() <= 2 * HALF * want.abs() + (HALF if rows > 8 else 2.0 ** -14) * size).all())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,hidden", [(4, 512), (8, 512)])
def test_single_block_over_selected_blocks(heads, hidden):
    g = seeded(heads)
    B, L = 2, 700
    blk = block(tk.SingleStreamBlock, hidden, heads).to(DEV)
    x, vec = randn(g, B, L, hidden, dtype=BF).to(DEV), randn(g, B, hidden, dtype=BF).to(DEV)
    ids = torch.arange(L, dtype=torch.float32, device=DEV).expand(B, L)[..., None]
    pe = tk.rope_table(ids[:1], [hidden // heads])
    with torch.no_grad():
        dense = blk(x, vec, pe)
        blk.sparse_keep = 11
        every = blk(x, vec, pe)
        # the same sums in another order of roundings: a few half steps of the attention, through one projection and a residual
        assert (every - dense).float().pow(2).mean().sqrt() <= 2 * HALF * dense.float().pow(2).mean().sqrt()
        blk.sparse_keep, blk.sparse_always = 4, 1
        blk.modulation.quantize()
        fused = blk(x, vec, pe)
        plain = copy.deepcopy(blk)
        plain.fused = False
        unfused = plain(x, vec, pe)
        assert (fused - dense).abs().max() > 0.01
        assert (fused - unfused).float().pow(2).mean().sqrt() <= 2 * HALF * unfused.float().pow(2).mean().sqrt()
        # one operator behind the other, those that are new from their plain statements on the CPU
        q, scale, _ = blk.modulation.lin.weight.unpack()
        mod = tk.linear_w4_torch(vec.cpu(), q.cpu(), scale.cpu(), None, blk.modulation.lin.bias.cpu(), in_activation="SiLU").to(DEV)[:, None].chunk(3, -1)
        y = blk.linear1(tk.layer_norm_modulation(x, mod[1], mod[0]))
        qh, kh, vh = y[..., :3 * hidden].view(B, L, 3, heads, -1).permute(2, 0, 3, 1, 4)
        qh, kh = tk.apply_rope(*blk.norm(qh, kh, vh), pe)
        lists = tk.select_blocks(qh, kh, 4, always=1)
        assert torch.equal(lists.cpu(), tk.select_blocks_torch(qh.cpu(), kh.cpu(), 4, 1))
        attn = tk.block_sparse_attention_torch(qh.cpu(), kh.cpu(), vh.cpu(), lists.cpu()).to(DEV)
        both = torch.cat((attn.transpose(1, 2).flatten(2), F.gelu(y[..., 3 * hidden:].float(), approximate="tanh").to(BF)), -1)
        want = x + mod[2] * blk.linear2(both)
    assert (fused - want).float().pow(2).mean().sqrt() <= 3 * HALF * want.float().pow(2).mean().sqrt()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 2])
def test_double_block_over_selected_blocks(B):
    g = seeded(B)
    hidden, heads, Lt, Li = 512, 4, 64, 400
    blk = block(tk.DoubleStreamBlock, hidden, heads, mlp_ratio=2.0, qkv_bias=True).to(DEV)
    img, txt, vec = randn(g, B, Li, hidden, dtype=BF).to(DEV), randn(g, B, Lt, hidden, dtype=BF).to(DEV), randn(g, B, hidden, dtype=BF).to(DEV)
    pe = tk.rope_table(torch.arange(Lt + Li, dtype=torch.float32, device=DEV)[None, :, None], [128])
    with torch.no_grad():
        dense = blk(img, txt, vec, pe)
        blk.sparse_keep = 8
        for a, b in zip(blk(img, txt, vec, pe), dense):
            assert (a - b).float().pow(2).mean().sqrt() <= 2 * HALF * b.float().pow(2).mean().sqrt()
        blk.sparse_keep, blk.sparse_always = 3, 1
        blk.img_mod.quantize(128)
        blk.txt_mod.quantize(32, True)
        fused = blk(img, txt, vec, pe)
        plain = copy.deepcopy(blk)
        plain.fused = False
        for a, b, d in zip(fused, plain(img, txt, vec, pe), dense):
            assert (a - d).abs().max() > 0.01
            assert (a - b).float().pow(2).mean().sqrt() <= 3 * HALF * b.float().pow(2).mean().sqrt()


@pytest.mark.gpu
def test_a_served_block_in_a_graph():
    g = seeded(9)
    hidden, heads, L = 512, 4, 300
    blk = block(tk.SingleStreamBlock, hidden, heads).to(DEV)
    blk.modulation.quantize()
    blk.sparse_keep = 2
    x, vec = randn(g, 1, L, hidden, dtype=BF).to(DEV), randn(g, 1, hidden, dtype=BF).to(DEV)
    pe = tk.rope_table(torch.arange(L, dtype=torch.float32, device=DEV)[None, :, None], [128])
    with torch.no_grad():
        blk(x, vec, pe)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = blk(x, vec, pe)
        for _ in range(3):
            x.copy_(randn(g, 1, L, hidden, dtype=BF))
            vec.copy_(randn(g, 1, hidden, dtype=BF))
            graph.replay()
            assert torch.equal(out, blk(x, vec, pe))
