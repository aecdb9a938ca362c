"""Projections of a block that are turned into ones with weights in 4 bits: they compute what the projection computed, or are refused."""
import math

import pytest
import torch

import triton_kernels as tk
from triton_kernels.modules import Linear, LinearGELU, LinearW4, Modulation
from util import DEV, randn, seeded

BF = torch.bfloat16
HALF = torch.finfo(BF).eps / 2


def parameters(g, lin):
    lin.weight.data, lin.bias.data = randn(g, *lin.weight.shape, std=0.1), randn(g, *lin.bias.shape)
    return lin


def formula(x, w4, bias):
    """x W^T + b in float64 with the weight that the numbers stand for, and how far sums in fp32 may be from it: K + 8 sums and products of numbers of at most
    s (16 + q + 16 + z) |x|, each good to 2^-23."""
    q, scale, zero = w4.weight.unpack()
    z = 8.0 if zero is None else zero.double()[..., None]
    by_group = q.double().unflatten(1, (-1, w4.group))
    w, reach = (((by_group + add) * scale.double()[..., None]).flatten(1) for add in (-z, 32 + z))
    return x.double() @ w.T + bias.double(), (x.shape[1] + 8) * 2.0 ** -23 * (x.double().abs() @ reach.T + bias.double().abs())


def test_a_projection_keeps_its_activation():
    g = seeded(1)
    assert LinearW4.from_linear(LinearGELU(64, 32)).activation == "GELU"
    assert all(LinearW4.from_linear(cls(64, 32)).activation == "" for cls in (Linear, torch.nn.Linear))
    assert LinearW4(64, 32).activation == "" and LinearW4(64, 32, activation="GELU").activation == "GELU"
    with pytest.raises(AssertionError):
        LinearW4(64, 32, activation="ReLU")
    # what is in the state is the same with and without
    a, b = LinearW4.from_linear(parameters(g, LinearGELU(64, 32))), LinearW4(64, 32, activation="GELU")
    b.load_state_dict(a.state_dict())
    assert all(torch.equal(s, t) for s, t in zip(a.state_dict().values(), b.state_dict().values()))


def test_projections_that_compute_something_else_are_refused():
    class Twice(Linear):
        def forward(self, input):
            return 2 * super().forward(input)

    hooked, early, patched = Linear(64, 32), torch.nn.Linear(64, 32), Linear(64, 32)
    hooked.register_forward_hook(lambda module, args, out: 2 * out)
    early.register_forward_pre_hook(lambda module, args: (2 * args[0],))
    patched.forward = lambda input: input
    normed = torch.nn.utils.parametrizations.weight_norm(torch.nn.Linear(64, 32))
    for lin in (Twice(64, 32), hooked, early, patched, normed, torch.nn.Identity(), LinearW4(64, 32)):
        with pytest.raises(AssertionError):
            LinearW4.from_linear(lin)
    modulation = Modulation(64, double=False)
    modulation.lin = Twice(64, 192)
    with pytest.raises(AssertionError):
        modulation.quantize()
    assert isinstance(modulation.lin, Twice)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,group,zeros", [(1, 64, False), (9, 32, True), (40, 128, True)])
def test_a_converted_projection_against_float64(rows, group, zeros):
    g = seeded(rows)
    lin = parameters(g, LinearGELU(256, 48)).to(BF)
    x = randn(g, rows, 256, dtype=BF)
    w4 = LinearW4.from_linear(lin, group, zeros)
    y, off = formula(x, w4, lin.bias.detach())
    want = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    # GELU's slope is at most 1.13, its exponential and reciprocal are good to 2^-20
    off = 1.13 * off + 2.0 ** -19 * want.abs()
    with torch.no_grad():
        got = w4.to(DEV)(x.to(DEV)).double().cpu()
    assert bool(((got - want).abs() <= off + HALF * (want.abs() + off)).all())
    assert (want - y).abs().max() > 0.1   # (without it the result is another)


@pytest.mark.gpu
def test_a_converted_projection_of_an_mlp():
    """Its first layer in 4 bits, the other as it is: the first layer's result is that of the operator with GELU."""
    g = seeded(5)
    mlp = tk.modules.blocks.MLP(128, 256).to(BF)
    x = randn(g, 2, 20, 128, dtype=BF).to(DEV)
    w = tk.quantize_w4(mlp[0].weight, 64).to(DEV)
    mlp[0] = LinearW4.from_linear(mlp[0])
    mlp.to(DEV)
    with torch.no_grad():
        hidden = tk.linear_w4(x, w, mlp[0].bias, activation="GELU")
        assert torch.equal(mlp[0](x), hidden) and torch.equal(mlp(x), mlp[2](hidden))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 12])
def test_a_modulation_whose_projection_has_an_activation(rows):
    g = seeded(rows)
    modulation = Modulation(128, double=False)
    modulation.lin = LinearW4.from_linear(parameters(g, LinearGELU(128, 384)))
    modulation.to(DEV)
    vec = randn(g, rows, 128, dtype=BF).to(DEV)
    with torch.no_grad():
        out, _ = modulation(vec)
        # (SiLU of its own rounds to bf16, on the way in it keeps 16 bits: one half step of every value apart)
        plain = modulation.lin(torch.nn.functional.silu(vec))
        got = torch.cat((out.shift, out.scale, out.gate), -1)[:, 0]
        size = torch.nn.functional.silu(vec).float().abs() @ modulation.lin.weight.dequantize().float().abs().T
    assert bool(((got.float() - plain.float()).abs() <= 1.13 * 2 * HALF * size + 2 * HALF * plain.float().abs()).all())


def _single(hidden=256, heads=4):
    torch.manual_seed(0)
    return tk.SingleStreamBlock(hidden, heads, mlp_ratio=2.0).to(BF)


def _double(hidden=256, heads=4):
    torch.manual_seed(0)
    return tk.DoubleStreamBlock(hidden, heads, mlp_ratio=2.0, qkv_bias=True).to(BF)


def _set(block, path, module):
    *at, last = path.split(".")
    for name in at:
        block = getattr(block, name)
    setattr(block, last, module)


@pytest.mark.gpu
@pytest.mark.parametrize("paths", [("linear1",), ("linear2",), ("linear1", "linear2", "modulation.lin")])
@pytest.mark.parametrize("keep", [None, 4])   # (4: every block, by way of their selection)
def test_single_block_with_projections_in_4_bits(paths, keep):
    """Beside the fused block whose weights are what the numbers stand for."""
    g = seeded(len(paths))
    block, plain = _single(), _single()
    _served(g, block, plain, paths)
    block.sparse_keep = plain.sparse_keep = keep
    x, vec = randn(g, 2, 200, 256, dtype=BF).to(DEV), randn(g, 2, 256, dtype=BF).to(DEV)
    pe = tk.rope_table(torch.arange(200, dtype=torch.float32, device=DEV)[None, :, None], [64])
    with torch.no_grad():
        got, want = block(x, vec, pe), plain(x, vec, pe)
    assert (got - want).float().pow(2).mean().sqrt() <= 3 * HALF * want.float().pow(2).mean().sqrt()


@pytest.mark.gpu
@pytest.mark.parametrize("paths", [("img_attn.qkv",), ("txt_attn.qkv",), ("img_attn.proj", "txt_attn.proj"), ("img_mlp.0",), ("txt_mlp.0",), ("img_mlp.2",), ("txt_mlp.2",),
                                   ("img_mod.lin", "txt_mod.lin", "img_attn.qkv", "txt_attn.qkv", "img_attn.proj", "txt_attn.proj", "img_mlp.0", "img_mlp.2", "txt_mlp.0", "txt_mlp.2")])
@pytest.mark.parametrize("B", [1, 2])
def test_double_block_with_projections_in_4_bits(paths, B):
    g = seeded(len(paths))
    block, plain = _double(), _double()
    _served(g, block, plain, paths)
    img, txt, vec = randn(g, B, 150, 256, dtype=BF).to(DEV), randn(g, B, 40, 256, dtype=BF).to(DEV), randn(g, B, 256, dtype=BF).to(DEV)
    pe = tk.rope_table(torch.arange(190, dtype=torch.float32, device=DEV)[None, :, None], [64])
    with torch.no_grad():
        for got, want in zip(block(img, txt, vec, pe), plain(img, txt, vec, pe)):
            assert (got - want).float().pow(2).mean().sqrt() <= 3 * HALF * want.float().pow(2).mean().sqrt()


def _served(g, block, plain, paths):
    """The projections at `paths`: in 4 bits with scales that are powers of two in `block`, whose weights bf16 holds as they are, and as such in `plain`."""
    for path in paths:
        lin = block.get_submodule(path)
        n, k = lin.weight.shape
        q, scale = torch.randint(0, 16, (n, k), generator=g), torch.full((n, k // 64), 2.0 ** -7, dtype=BF)
        w4 = LinearW4.from_linear(lin, 64)
        w = tk.pack_w4(q, scale)
        w4.packed, w4.scale = w.packed, w.scale
        _set(block, path, w4)
        plain.get_submodule(path).weight.data = ((q - 8) * 2.0 ** -7).to(BF)
    block.to(DEV), plain.to(DEV)


@pytest.mark.gpu
def test_a_block_wholly_in_4_bits_in_a_graph():
    g = seeded(6)
    block, plain = _double(), _double()
    _served(g, block, plain, ("img_mod.lin", "txt_mod.lin", "img_attn.qkv", "txt_attn.qkv", "img_attn.proj", "txt_attn.proj", "img_mlp.0", "img_mlp.2", "txt_mlp.0", "txt_mlp.2"))
    img, txt, vec = randn(g, 1, 150, 256, dtype=BF).to(DEV), randn(g, 1, 40, 256, dtype=BF).to(DEV), randn(g, 1, 256, dtype=BF).to(DEV)
    pe = tk.rope_table(torch.arange(190, dtype=torch.float32, device=DEV)[None, :, None], [64])
    with torch.no_grad():
        block(img, txt, vec, pe)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(img, txt, vec, pe)
        for _ in range(3):
            img.copy_(randn(g, 1, 150, 256, dtype=BF))
            vec.copy_(randn(g, 1, 256, dtype=BF))
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, block(img, txt, vec, pe)))


def test_which_blocks_run_fused():
    """On the CPU: a block with a projection in 4 bits, beside its modulations, takes its operators one at a time."""
    for make, mods, rest in ((_single, ("modulation.lin",), ("linear1", "linear2")),
                             (_double, ("img_mod.lin", "txt_mod.lin"), ("img_attn.qkv", "txt_attn.qkv", "img_attn.proj", "txt_attn.proj", "img_mlp.0", "img_mlp.2", "txt_mlp.0", "txt_mlp.2"))):
        for path in mods + rest:
            block = make()
            assert block._projections_in_4_bits() is False
            _set(block, path, LinearW4.from_linear(block.get_submodule(path)))
            assert block._projections_in_4_bits() is (path in rest)


@pytest.mark.gpu
def test_blocks_with_projections_in_4_bits_in_code_that_is_traced():
    torch._dynamo.reset()
    g = seeded(7)
    single, double = _single().to(DEV), _double().to(DEV)
    x, vec = randn(g, 1, 190, 256, dtype=BF).to(DEV), randn(g, 1, 256, dtype=BF).to(DEV)
    pe = tk.rope_table(torch.arange(190, dtype=torch.float32, device=DEV)[None, :, None], [64])
    single.linear1, double.img_mlp[0] = LinearW4.from_linear(single.linear1), LinearW4.from_linear(double.img_mlp[0])
    with torch.no_grad():
        for keep in (None, 2):
            single.sparse_keep = double.sparse_keep = keep
            assert torch.equal(torch.compile(single, backend="eager")(x, vec, pe), single(x, vec, pe))
            args = x[:, 40:], x[:, :40], vec, pe
            assert all(torch.equal(a, b) for a, b in zip(torch.compile(double, backend="eager")(*args), double(*args)))
    torch._dynamo.reset()
