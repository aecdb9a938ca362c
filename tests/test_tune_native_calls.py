"""layer_norm, apply_rope_nd, rope_table and linear_lora in native code (csrc/torch_ops.cpp) against the Python launchers of the same operators, over the
forms they accept and with what autograd can do to their saved tensors, and the calls that they leave to the launchers."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwad

import triton_kernels as tk
from triton_kernels import _native as nv
from util import DEV, randn, seeded

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
AXES = (16, 24, 24)


class _Refuses:
    """Native calls that take nothing: every operator goes through its Python launcher."""

    def __getattr__(self, name):
        return lambda *args: None


class _Counts:
    """Native calls that note whether they took what they were given."""

    def __init__(self):
        self.ops, self.took = nv.ops(), []

    def __getattr__(self, name):
        def call(*args):
            out = getattr(self.ops, name)(*args)
            self.took.append(out is not None)
            return out
        return call


def launcher(monkeypatch, fn, *args, **kw):
    with monkeypatch.context() as m:
        m.setattr(nv, "ops", lambda: _Refuses())
        return fn(*args, **kw)


def took(monkeypatch, fn, *args, **kw):
    """Whether the native call of an operator, called once, took it."""
    counts = _Counts()
    with monkeypatch.context() as m:
        m.setattr(nv, "ops", lambda: counts)
        fn(*args, **kw)
    assert len(counts.took) == 1
    return counts.took[0]


def same(a, b):
    assert len(a) == len(b)
    for s, t in zip(a, b):
        assert (s is None) == (t is None)
        if s is not None:
            assert s.dtype == t.dtype and s.shape == t.shape and s.stride() == t.stride() and torch.equal(s.nan_to_num(7.0), t.nan_to_num(7.0))


def norm_step(x, w, b, dy, plus_one=False, wanted="xwb", hooks=None):
    leaves = {n: t.detach().requires_grad_(n in wanted) for n, t in zip("xwb", (x, w, b)) if t is not None}
    if hooks is None:
        y = tk.layer_norm(leaves["x"], leaves.get("w"), leaves.get("b"), 1e-5, plus_one=plus_one)
    else:
        with hooks:
            y = tk.layer_norm(leaves["x"], leaves.get("w"), leaves.get("b"), 1e-5, plus_one=plus_one)
    wanted = [leaves[n] for n in wanted if n in leaves]
    return [y.detach(), *(torch.autograd.grad(y, wanted, dy) if wanted else ())]


def rope_step(q, k, ids, dq, dk, hooks=None, wanted="qk"):
    q = q.detach().requires_grad_("q" in wanted)
    k = k if k is None else k.detach().requires_grad_("k" in wanted)
    if hooks is None:
        out = tk.apply_rope_nd(q, k, ids, AXES)
    else:
        with hooks:
            out = tk.apply_rope_nd(q, k, ids, AXES)
    leaves = [t for t in (q, k) if t is not None and t.requires_grad]
    outs = [(y, d) for y, d in zip(out, (dq, dk)) if y is not None and y.requires_grad]
    return [t if t is None else t.detach() for t in out] + list(torch.autograd.grad([y for y, _ in outs], leaves, [d for _, d in outs], allow_unused=True) if leaves else ())


def test_what_is_not_on_a_gpu_is_left_to_the_launchers():
    ops, x, ids = nv.ops(), torch.ones(2, 2, 4, 64), torch.zeros(4, 3)
    assert ops.layer_norm(x, None, None, 1e-5, False) is None
    assert ops.apply_rope_nd(x, x, ids, AXES, 1e4) is None and ops.rope_table(ids, AXES, 1e4) is None
    b = x.bfloat16()
    assert ops.linear_lora(b, torch.ones(8, 64, dtype=BF), None, torch.ones(1, 2, 64, dtype=BF), torch.ones(1, 8, 2, dtype=BF), torch.zeros(2, dtype=torch.int32), None, 0) is None
    for bad in (None, 3, "x", [x]):
        assert ops.layer_norm(bad, None, None, 1e-5, False) is None and ops.layer_norm(x, bad if bad is not None else 3, None, 1e-5, False) is None
        assert ops.apply_rope_nd(bad, x, ids, AXES, 1e4) is None and ops.apply_rope_nd(x, x, bad, AXES, 1e4) is None and ops.rope_table(ids, bad, 1e4) is None
        assert ops.linear_lora(bad, b, None, b, b, b, None, 0) is None
    for args, name in (((x,), "layer_norm"), ((x,), "apply_rope_nd"), ((), "rope_table"), ((x, x), "linear_lora")):
        with pytest.raises(RuntimeError, match="arguments"):
            getattr(ops, name)(*args)


@gpu
@pytest.mark.parametrize("dtype,w_dtype", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
def test_layer_norm(monkeypatch, dtype, w_dtype):
    g = seeded(1)
    base = randn(g, 3, 4, 5, 128, dtype=dtype).to(DEV)
    wide = randn(g, 2, 6, 768, dtype=dtype).to(DEV)
    odd = randn(g, 901, dtype=dtype).to(DEV)
    views = [base, base[0, 0, 0], base[1], base.permute(2, 0, 1, 3), base.transpose(1, 2)[::2], wide[..., 256:512], base[..., :100], base[..., 1:51], base[:, :, :1].expand(3, 4, 7, 128),
             odd[1:], odd[3:3 + 5 * 33].view(5, 33), base[..., ::2], base[:0], base[:, :0], base[..., :1], base.transpose(0, 3)]
    for i, x in enumerate(views):
        n, lead = x.shape[-1], x.shape[0]
        dy = randn(g, *x.shape, dtype=dtype).to(DEV)
        shared = [randn(g, n, dtype=w_dtype).to(DEV) for _ in range(2)]
        each = [randn(g, lead, *(1,) * (x.dim() - 2), 2 * n, dtype=w_dtype).to(DEV)[..., n:] for _ in range(2)] if x.dim() > 1 else shared
        for w, b in (shared, (None, None), (shared[0], None), (None, shared[1]), each, (each[0], None), (each[0], shared[1]), (shared[0].view(*(1,) * i, n)[(0,) * (i - 1)] if i > 1 else shared[0], None)):
            for wanted in ("xwb", "x", "wb", "b", ""):
                args = (x, w, b, dy, i % 2 == 1, wanted)
                same(norm_step(*args), launcher(monkeypatch, norm_step, *args))
    x = base
    assert took(monkeypatch, tk.layer_norm, x, torch.ones(128, dtype=dtype, device=DEV), None)
    assert not took(monkeypatch, tk.layer_norm, x[..., ::2])


@gpu
def test_layer_norm_gives_what_saved_tensor_hooks_give_back(monkeypatch):
    """Saved tensors on the CPU and back, as copies of another layout, and replaced by others."""
    g = seeded(2)
    x, dy, w, b = randn(g, 2, 9, 256, dtype=BF).to(DEV), randn(g, 2, 9, 256, dtype=BF).to(DEV), randn(g, 256, dtype=BF).to(DEV), randn(g, 256, dtype=BF).to(DEV)
    want = norm_step(x, w, b, dy)
    same(norm_step(x, w, b, dy, hooks=torch.autograd.graph.save_on_cpu()), want)

    def spread(t):
        return torch.stack((t, t), -1)[..., 0]                                        # the same values, two elements apart

    same(norm_step(x, w, b, dy, hooks=torch.autograd.graph.saved_tensors_hooks(spread, lambda t: t)), want)
    for call in (norm_step, lambda *a, **k: launcher(monkeypatch, norm_step, *a, **k)):
        with pytest.raises(RuntimeError, match="other sizes"):
            call(x, w, b, dy, hooks=torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[..., :-1]))
        with pytest.raises(RuntimeError, match="devices|GPU"):
            call(x, w, b, dy, hooks=torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu() if t.dim() == 1 or t.shape[0] == 1 else t))
    xl = x.clone().requires_grad_(True)
    y = tk.layer_norm(xl * 1.0, w, b)
    kept = xl * 1.0
    z = tk.layer_norm(kept, w, b)
    kept.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        z.sum().backward()


@gpu
def test_layer_norm_is_differentiated_once(monkeypatch):
    """A gradient of its gradients is an error wherever it comes from: from dy, from x or from the weight."""
    g = seeded(8)
    x, w, b, dy = (randn(g, *shape).to(DEV).requires_grad_(True) for shape in ((2, 9, 64), (64,), (64,), (2, 9, 64)))

    def both(fn):
        fn()
        launcher(monkeypatch, fn)

    def twice(inputs, weight, source, d):
        grads = torch.autograd.grad(tk.layer_norm(x if "x" in inputs else x.detach(), weight, b), [t for n, t in (("x", x), ("w", w), ("b", b)) if n in inputs], d, create_graph=True)
        for t in grads:
            assert t.requires_grad
            with pytest.raises(RuntimeError, match="differentiated once only"):
                torch.autograd.grad(t.sum(), source, retain_graph=True)

    both(lambda: twice("xwb", w, x, dy))
    both(lambda: twice("xw", w, w, dy.detach()))
    both(lambda: twice("xb", w.detach(), dy, dy))
    both(lambda: twice("x", None, x, dy.detach()))
    both(lambda: twice("b", None, dy, dy))
    plain = norm_step(x, w, b, dy.detach())
    again = torch.autograd.grad(tk.layer_norm(x, w, b, 1e-5), (x, w, b), dy.detach(), create_graph=True)
    same([t.detach() for t in again], plain[1:])


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_apply_rope_nd_and_rope_table(monkeypatch, dtype):
    g = seeded(3)
    x = randn(g, 2, 7, 3, 5, 64, dtype=dtype).to(DEV)                     # [B, L, 3, H, D], a fused projection
    q, k = x[:, :, 0].transpose(1, 2), x[:, :, 1, :2].transpose(1, 2)
    odd = randn(g, 2 * 5 * 7 * 64 + 1, dtype=dtype).to(DEV)[1:].view(2, 5, 7, 64)
    shifted = torch.randint(-40, 40, (2, 7, 6), generator=g).to(DEV)
    for kind in (F32, torch.float64, torch.int32, torch.int64, torch.int16, BF):
        for ids in (shifted[..., :3].to(kind), shifted.to(kind)[..., ::2], shifted[0, :, 3:].to(kind), shifted[:1, :, :3].to(kind), shifted[:1, :, :3].to(kind).expand(2, 7, 3)):
            for a, b in ((q, k), (odd, q.contiguous()), (q, None), (q[:, :1].expand(2, 4, 7, 64), k), (q.flip(3)[..., ::1], q.transpose(2, 3).contiguous().transpose(2, 3))):
                dq, dk = randn(g, *a.shape, dtype=dtype).to(DEV), None if b is None else randn(g, *b.shape, dtype=dtype).to(DEV)
                same(rope_step(a, b, ids, dq, dk), launcher(monkeypatch, rope_step, a, b, ids, dq, dk))
            for wanted in ("q", "k", ""):
                args = (q, k, ids, torch.ones_like(q), torch.ones_like(k), None, wanted)
                same(rope_step(*args), launcher(monkeypatch, rope_step, *args))
            for theta in (10000, 500.0):
                same([tk.rope_table(ids, list(AXES), theta)], [launcher(monkeypatch, tk.rope_table, ids, AXES, theta)])
    assert took(monkeypatch, tk.apply_rope_nd, q, k, shifted[..., :3], AXES) and took(monkeypatch, tk.rope_table, shifted[..., :3], AXES)
    assert not took(monkeypatch, tk.apply_rope_nd, q, k, shifted[..., :3].short(), AXES)


@gpu
def test_apply_rope_nd_with_hooks_and_ids_changed_in_between(monkeypatch):
    g = seeded(4)
    q, k, ids = randn(g, 2, 3, 6, 64).to(DEV), randn(g, 2, 1, 6, 64).to(DEV), torch.randint(0, 90, (2, 6, 3), generator=g).to(DEV)
    dq, dk = randn(g, *q.shape).to(DEV), randn(g, *k.shape).to(DEV)
    want = rope_step(q, k, ids, dq, dk)
    same(rope_step(q, k, ids, dq, dk, torch.autograd.graph.save_on_cpu()), want)
    same(rope_step(q, k, ids, dq, dk, torch.autograd.graph.saved_tensors_hooks(lambda t: t.double().transpose(0, 1).contiguous(), lambda t: t.transpose(0, 1))), want)
    for call in (rope_step, lambda *a: launcher(monkeypatch, rope_step, *a)):
        with pytest.raises((RuntimeError, AssertionError)):
            call(q, k, ids, dq, dk, torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:, :-1]))
    a = q.clone().requires_grad_(True)
    y, _ = tk.apply_rope_nd(a, None, ids, AXES)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@gpu
def test_linear_lora(monkeypatch):
    g = seeded(5)
    wide = randn(g, 4, 30, 600, dtype=BF).to(DEV)
    weights, bias = randn(g, 200, 600, dtype=BF).to(DEV), randn(g, 200, dtype=BF).to(DEV)
    a, b, s = randn(g, 3, 16, 600, dtype=BF).to(DEV), randn(g, 3, 200, 16, dtype=BF).to(DEV), torch.rand(3, generator=g).to(DEV)
    by_request, by_row = torch.tensor([0, 2, -1, 1], device=DEV), torch.randint(-2, 5, (4, 30), generator=g).to(DEV)
    for lo, hi in ((0, 600), (8, 264), (1, 257), (0, 63)):
        x, w, la = wide[..., lo:hi], weights[:, lo:hi], a[..., lo:hi]
        for xs, ad in ((x, by_request), (x, by_row), (x, by_request.int()), (x, by_row.int()), (x, by_row.short()), (x, by_request[1]), (x[:, :1], by_request), (x[2, 0], by_row[0, 0]),
                       (x[0, :1].expand(30, hi - lo), by_row[0]), (x.transpose(0, 1), by_row.T), (x[:, ::2], by_row[:, ::2]), (x[:0], by_request[:0])):
            for lora_a, lora_b, scaling, act in ((la.contiguous(), b, s, ""), (la, b, None, "GELU"), (la.contiguous(), b.transpose(1, 2).contiguous().transpose(1, 2), s.double(), "")):
                for bb in (None, bias, bias.float()):
                    args = (xs, w, bb, lora_a, lora_b, ad, scaling, act)
                    same([tk.linear_lora(*args)], [launcher(monkeypatch, tk.linear_lora, *args)])
    assert took(monkeypatch, tk.linear_lora, wide, weights, bias, a, b, by_request, s) and not took(monkeypatch, tk.linear_lora, wide, weights, bias, a, b, by_row.short(), s)
    big = randn(g, 64, 16384, dtype=BF, std=0.01).to(DEV), randn(g, 2048, 16384, dtype=BF, std=0.01).to(DEV), None, randn(g, 2, 8, 16384, dtype=BF, std=0.01).to(DEV), randn(g, 2, 2048, 8, dtype=BF).to(DEV), torch.zeros(64, dtype=torch.int64, device=DEV)
    same([tk.linear_lora(*big)], [launcher(monkeypatch, tk.linear_lora, *big)])     # K in parts: the workspace holds them


@gpu
def test_what_transforms_see():
    """Forward-mode derivatives and vmap are refused, as by the other operators; a subclass comes through the launchers."""
    x, ids = torch.randn(2, 3, 4, 64, device=DEV), torch.zeros(4, 3, device=DEV)
    for fn in (lambda t: tk.layer_norm(t), lambda t: tk.apply_rope_nd(t, t, ids, AXES)[0]):
        with fwad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            fn(fwad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.vmap(fn)(x[None])

    class Sub(torch.Tensor):
        pass

    assert torch.equal(torch.Tensor(tk.layer_norm(x.as_subclass(Sub)).as_subclass(torch.Tensor)), tk.layer_norm(x))
    p = torch.nn.Parameter(torch.ones(64, device=DEV))
    tk.layer_norm(x, p).sum().backward()
    assert p.grad is not None


@gpu
def test_calls_from_threads_on_streams_of_their_own():
    g = seeded(6)
    x, w, b, dy = randn(g, 2, 65, 768, dtype=BF).to(DEV), randn(g, 768, dtype=BF).to(DEV), randn(g, 768, dtype=BF).to(DEV), randn(g, 2, 65, 768, dtype=BF).to(DEV)
    weights, la, lb = randn(g, 96, 768, dtype=BF).to(DEV), randn(g, 2, 8, 768, dtype=BF).to(DEV), randn(g, 2, 96, 8, dtype=BF).to(DEV)
    ad = torch.tensor([1, 0], device=DEV)
    want = norm_step(x, w, b, dy) + [tk.linear_lora(x, weights, None, la, lb, ad)]
    torch.cuda.synchronize()
    failed = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                got = norm_step(x, w, b, dy) + [tk.linear_lora(x, weights, None, la, lb, ad)]
                stream.synchronize()
                if not all(torch.equal(s, t) for s, t in zip(got, want)):
                    failed.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@gpu
def test_inference_mode_one_row_and_numbers_of_no_adapter(monkeypatch):
    g = seeded(9)
    x, w, ids = randn(g, 2, 3, 4, 64, dtype=BF).to(DEV), randn(g, 64, dtype=BF).to(DEV), torch.randint(0, 9, (4, 3), generator=g).to(DEV)
    weights, la, lb = randn(g, 40, 64, dtype=BF).to(DEV), randn(g, 2, 8, 64, dtype=BF).to(DEV), randn(g, 2, 40, 8, dtype=BF).to(DEV)
    none = torch.tensor([2 ** 40, -2 ** 63], device=DEV)
    calls = (lambda: tk.layer_norm(x, w), lambda: tk.layer_norm(x[0, 0, 0], w), lambda: tk.apply_rope_nd(x, None, ids, AXES)[0], lambda: tk.rope_table(ids, AXES),
             lambda: tk.linear_lora(x, weights, None, la, lb, none), lambda: tk.linear_lora(x[0, 0, 0], weights, None, la, lb, none[0] * 0 + 1))
    for call in calls:
        want = call()
        with torch.inference_mode():
            assert torch.equal(call(), want)
        assert torch.equal(launcher(monkeypatch, call), want)
    assert torch.equal(calls[4](), tk.linear(x, weights, None))


@gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_under_activation_checkpoints(monkeypatch, reentrant):
    from torch.utils.checkpoint import checkpoint

    g = seeded(10)
    x, w = randn(g, 2, 6, 64, dtype=BF).to(DEV).requires_grad_(True), randn(g, 64, dtype=BF).to(DEV).requires_grad_(True)
    ids = torch.randint(0, 9, (6, 3), generator=g).to(DEV)

    def block(x, w):
        q, k = tk.apply_rope_nd(tk.layer_norm(x, w, w).unsqueeze(1), tk.layer_norm(x, None, w).unsqueeze(1), ids, AXES)
        return (q * k).float().sum()

    def both():
        grads = []
        for y in (block(x, w), checkpoint(block, x, w, use_reentrant=reentrant)):
            x.grad = w.grad = None
            y.backward()
            grads.append((x.grad, w.grad))
        same(*grads)

    both()
    launcher(monkeypatch, both)
