"""The operators called from code that torch.compile traces: a graph break each, and the results and gradients of the plain call."""
import pytest
import torch

import triton_kernels as tk
from triton_kernels import testing as cfg
from util import DEV, randn, seeded

BF = torch.bfloat16
AXES = (16, 24, 24)


@pytest.fixture(autouse=True)
def fresh():
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


def run(fn, args, dys, backend=None):
    leaves = [t.clone().requires_grad_(t.is_floating_point()) if isinstance(t, torch.Tensor) else t for t in args]
    outs = fn(*leaves) if backend is None else torch.compile(fn, backend=backend)(*leaves)
    outs = outs if isinstance(outs, tuple) else (outs,)
    wanted = [t for t in leaves if isinstance(t, torch.Tensor) and t.requires_grad]
    if not any(t.requires_grad for t in outs):
        return [t.detach() for t in outs]
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs, wanted, [dys(t) for t in outs], allow_unused=True))


CASES = {
    "layer_norm": lambda x, w, b, q, ids: ((lambda x, w, b: tk.layer_norm(x * 1.0, w, b, 1e-6, plus_one=True) + 0.0), (x, w, b)),
    "layer_norm_fp32_bias": lambda x, w, b, q, ids: ((lambda x, w, b: tk.layer_norm(x, w, b.float()) * 1.0), (x, w, b)),
    "apply_rope_nd": lambda x, w, b, q, ids: ((lambda q, k: tuple(t * 1.0 for t in tk.apply_rope_nd(q, k, ids, AXES))), (q, q[:, :1])),
    "apply_rope_nd_q": lambda x, w, b, q, ids: ((lambda q: tk.apply_rope_nd(q * 1.0, None, ids, AXES)[0]), (q,)),
    "rms_norm": lambda x, w, b, q, ids: ((lambda x, w: tk.rms_norm(x * 1.0, w) * 1.0), (x, w)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("name", CASES)
def test_operators_with_gradients(name, backend):
    g = seeded(1)
    x, w, b, q = randn(g, 2, 9, 64, dtype=BF).to(DEV), randn(g, 64, dtype=BF).to(DEV), randn(g, 64, dtype=BF).to(DEV), randn(g, 2, 3, 9, 64, dtype=BF).to(DEV)
    fn, args = CASES[name](x, w, b, q, torch.randint(0, 30, (9, 3), generator=g).to(DEV))
    dys = lambda t: torch.ones_like(t) * 0.5  # noqa: E731
    for got, want in zip(run(fn, args, dys, backend), run(fn, args, dys)):
        assert (got is None) == (want is None) and (got is None or torch.equal(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_operators_of_inference(backend):
    g = seeded(2)
    x, w, b = randn(g, 2, 9, 64, dtype=BF).to(DEV), randn(g, 40, 64, dtype=BF).to(DEV), randn(g, 40, dtype=BF).to(DEV)
    la, lb, s, ad = randn(g, 2, 8, 64, dtype=BF).to(DEV), randn(g, 2, 40, 8, dtype=BF).to(DEV), torch.rand(2, generator=g).to(DEV), torch.tensor([1, -1], device=DEV)
    q, ids = randn(g, 2, 3, 9, 64, dtype=BF).to(DEV), torch.randint(0, 30, (9, 3), generator=g).to(DEV)
    mod = randn(g, 2, 1, 128, dtype=BF).to(DEV)
    calls = (lambda x: tk.linear_lora(x * 1.0, w, b, la, lb, ad, s, activation="GELU") * 2.0, lambda x: tk.linear_lora(x, w, None, la, lb, ad.short()), lambda x: tk.rope_table(ids, list(AXES)) + x.float().sum() * 0,
             lambda x: tk.EmbedND(64, 10000, list(AXES))(ids) + x.float().sum() * 0, lambda x: tk.linear(x * 1.0, w, b) * 2.0, lambda x: tk.linear_into(x, w, b),
             lambda x: tk.layer_norm_modulation(x, mod[..., :64], mod[..., 64:]) * 1.0, lambda x: tk.scaled_dot_product_attention(q + x.sum() * 0, q, q) * 1.0,
             lambda x: tk.attention_into(q, q, q, torch.empty_like(q)) * 1.0, lambda x: tk.apply_rope(q, q, tk.rope_table(ids, AXES))[1] * 1.0, lambda x: tk.qkv_prep(q, q, q, pe=tk.rope_table(ids, AXES))[2] * 1.0)
    for fn in calls:
        with torch.no_grad():
            torch._dynamo.reset()
            compiled = torch.compile(fn, backend=backend)
            for t in (x, x * 2, x[:, :5] if fn is calls[4] else x):
                want = fn(t)
                assert torch.equal(compiled(t), want)


@pytest.mark.gpu
def test_modules():
    """A module of one's own around them, trained a step."""
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.proj, self.qk = tk.LayerNorm(64), torch.nn.Linear(64, 192), tk.RMSNorm(64)

        def forward(self, x, ids):
            q, k, v = self.proj(self.norm(x)).unflatten(-1, (3, 1, 64)).permute(2, 0, 3, 1, 4)
            q, k = tk.apply_rope_nd(self.qk(q), k, ids, AXES)
            return (torch.softmax((q.unsqueeze(3) * k.unsqueeze(2)).sum(-1) / 8, -1).unsqueeze(-1) * v.unsqueeze(2)).sum(3)

    g = seeded(3)
    torch.manual_seed(0)
    block = Block().to(DEV)
    x, ids = randn(g, 2, 11, 64).to(DEV), torch.randint(0, 30, (11, 3), generator=g).to(DEV)
    grads = []
    for fn in (block, torch.compile(block, backend="eager")):
        block.zero_grad()
        fn(x, ids).square().sum().backward()
        grads.append([p.grad.clone() for p in block.parameters()])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_blocks():
    heads, hidden = 4, 512
    x, vec, pe, sd = cfg.config5_block("cpu", n_txt=32, grid=8, hidden=hidden, heads=heads)
    x, vec, pe = x.to(DEV), vec.to(DEV), pe.to(DEV)
    single = tk.SingleStreamBlock(hidden, heads).to(BF).to(DEV)
    single.load_state_dict(sd)
    torch.manual_seed(1)
    double = tk.DoubleStreamBlock(hidden, heads, mlp_ratio=4.0, qkv_bias=True).to(BF).to(DEV)
    with torch.no_grad():
        for fused in (True, False):
            single.fused = double.fused = fused
            torch._dynamo.reset()
            want = single(x, vec, pe)
            assert torch.equal(torch.compile(single, backend="eager")(x, vec, pe), want)
            assert torch.equal(torch.compile(lambda x: single(x * 1.0, vec, pe) * 1.0, backend="eager")(x), want)
            for got, ref in zip(torch.compile(double, backend="eager")(x[:, 32:], x[:, :32], vec, pe), double(x[:, 32:], x[:, :32], vec, pe)):
                assert torch.equal(got, ref)
