"""Operators around a transformer block that is fine-tuned or serves many requests, as measurable cases: layer norm with
its gradients, rotation by positions of several axes, and projections with a low-rank adapter of each request's own.

`own` False: `run` computes them from elementary torch operations in 32 bits (angles in 64), rounded once at the end;
True: it makes the calls of the package. Imported with the repository's root as the working folder.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "triton-kernels_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# One large image in a batch of three, in tokens: the most rows of a norm or a projection.
MOST_ROWS = 3 * 4336
# Values of q and k of the longest video: drawn rotations stay at or below it.
MOST_ROTATED = 2 * 24 * 32760 * 128
# Multiplications of the largest projection with adapters.
MOST_PRODUCTS = MOST_ROWS * 3072 * 12288


def listed():
    return [
        # Training step of the adaLN norm of a block at one 1024 x 1024 image and its text: scale and shift of the one batch element.
        {"name": "norm_train_4608", "kind": "norm", "dtype": "bf16", "batch": 1, "tokens": 4608, "width": 3072, "weights": "modulation", "train": True},
        # The same on a batch of three images: the largest; the gradients of scale and shift are sums over each image's own rows.
        {"name": "norm_train_b3_4336", "kind": "norm", "dtype": "bf16", "batch": 3, "tokens": 4336, "width": 3072, "weights": "modulation", "train": True},
        # Training step of a text encoder's norm, in float32, with a weight and a bias that all rows share; odd row count.
        {"name": "norm_train_fp32_1001", "kind": "norm", "dtype": "fp32", "batch": 4, "tokens": 1001, "width": 1024, "weights": "affine", "train": True},
        # One short prompt through such a norm, forward only: the smallest call.
        {"name": "norm_77", "kind": "norm", "dtype": "bf16", "batch": 1, "tokens": 77, "width": 768, "weights": "affine", "train": False},
        # q and k of a video of 21 latent frames of 30 x 52 patches, read where the fused projection leaves them: the largest rotation.
        {"name": "rope_video_32760", "kind": "rope", "dtype": "bf16", "batch": 1, "heads": 24, "kv_heads": 24, "text": 0, "frames": 21, "height": 30, "width": 52,
         "axes": "16,56,56", "far": 0, "train": False},
        # Training step on two requests' images with text in front, fewer heads of k than of q, float32.
        {"name": "rope_train_1107", "kind": "rope", "dtype": "fp32", "batch": 2, "heads": 16, "kv_heads": 4, "text": 77, "frames": 1, "height": 32, "width": 32 + 1,
         "axes": "32,48,48", "far": 0, "train": True},
        # One new token of each of four streams, far along the time axis.
        {"name": "rope_token_far", "kind": "rope", "dtype": "bf16", "batch": 4, "heads": 24, "kv_heads": 8, "text": 0, "frames": 1, "height": 1, "width": 1,
         "axes": "16,56,56", "far": 1000000, "train": False},
        # The rotation table of a 1024 x 1024 image and its text, as the blocks take it.
        {"name": "rope_table_4608", "kind": "table", "batch": 1, "text": 512, "frames": 1, "height": 64, "width": 64, "axes": "16,56,56", "far": 0},
        # The mlp's first projection for three requests of one large image each, an adapter each: the largest product.
        {"name": "lora_b3_4336_gelu", "kind": "lora", "requests": 3, "rows": 4336, "in": 3072, "out": 12288, "rank": 16, "adapters": 8, "act": "GELU"},
        # The q, k and v projection of two requests of 2304 tokens, adapters of rank 64.
        {"name": "lora_b2_2304", "kind": "lora", "requests": 2, "rows": 2304, "in": 3072, "out": 9216, "rank": 64, "adapters": 4, "act": ""},
        # Rows of many requests packed one behind the other, an adapter by row; ranks of 32.
        {"name": "lora_packed_517", "kind": "lora", "requests": 517, "rows": 1, "in": 2048, "out": 2048, "rank": 32, "adapters": 16, "act": ""},
        # The modulation projection of the conditioning vectors of six requests: the smallest product.
        {"name": "lora_rows_6", "kind": "lora", "requests": 6, "rows": 1, "in": 1024, "out": 6144, "rank": 16, "adapters": 32, "act": ""},
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "rope", "rope", "table", "lora", "lora", "lora"])
    if kind == "norm":
        # widths that fill 16-byte vectors, and now and then any width
        width = 8 * _log_int(rng, 8, 1024) if rng.random() < 0.8 else _log_int(rng, 33, 5000)
        batch = rng.randint(1, 4)
        tokens = _log_int(rng, 1, max(1, MOST_ROWS * 3072 // (width * batch * 2)))
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp32"]), "batch": batch, "tokens": min(tokens, 16384), "width": width,
                "weights": rng.choice(["modulation", "affine", "none"]), "train": rng.random() < 0.7}
    if kind in ("rope", "table"):
        axes = rng.choice(["16,56,56", "32,48,48", "64", "32,32", "44,42,42", "8,24,32", "16,16,32,64", "24,12,12", "64,96,96"])
        side = _log_int(rng, 1, 128)
        frames = rng.choice([1, 1, _log_int(rng, 1, 32)])
        case = {"kind": kind, "batch": rng.randint(1, 4), "text": rng.choice([0, 0, 1, 77, 512]), "frames": frames, "height": side, "width": _log_int(rng, 1, 128),
                "axes": axes, "far": rng.choice([0, 0, 1000, 1000000])}
        if kind == "table":
            while case["batch"] * (case["text"] + case["frames"] * case["height"] * case["width"]) > 2 * 32760:
                case["height"] = (case["height"] + 1) // 2
            return case
        case |= {"dtype": rng.choice(["bf16", "bf16", "fp32"]), "heads": rng.choice([1, 8, 16, 24, 32]), "train": rng.random() < 0.4}
        case["kv_heads"] = rng.choice([case["heads"], max(1, case["heads"] // 4), 1])
        dim = sum(map(int, axes.split(",")))
        most = MOST_ROTATED // (4 if case["train"] else 2)
        while case["batch"] * (case["heads"] + case["kv_heads"]) * (case["text"] + case["frames"] * case["height"] * case["width"]) * dim > most:
            case["height"] = (case["height"] + 1) // 2
            if case["height"] == 1:
                case["frames"] = case["batch"] = 1
        return case
    # projections: widths of a model, of any multiple of 8, outputs of any number
    k = rng.choice([768, 1024, 1536, 3072, 4096, 8 * _log_int(rng, 8, 768)])
    n = rng.choice([k, 3 * k, 4 * k, 6 * k, _log_int(rng, 64, 12288)])
    rows = _log_int(rng, 1, max(1, min(MOST_ROWS, MOST_PRODUCTS // (k * n) // 2)))
    by_row = rng.random() < 0.4
    requests = min(rows, 1024) if by_row else rng.randint(1, 8)
    return {"kind": kind, "requests": requests, "rows": 1 if by_row else max(1, rows // requests), "in": k, "out": n, "rank": rng.choice([4, 8, 12, 16, 32, 64, 128]),
            "adapters": rng.choice([1, 2, 5, 16, 32]), "act": rng.choice(["", "", "GELU"])}


class _Inputs:
    """Seeded values, drawn on the GPU in float32."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(shape, generator=self.g, device="cuda").mul_(std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def whole(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda")


def _axes(case):
    return [int(a) for a in case["axes"].split(",")]


def _ids(case, inputs):
    """[batch, tokens, axes]: text at position 0, then the raster of every frame, which begins at a place of its own in every batch element, as a
    crop of a larger picture does; a stream that is far along starts at an offset on the first axis as well. One axis: places in the sequence;
    two: height and width; four: another axis in front that is 0 for images."""
    n = len(_axes(case))
    t, h, w = (torch.arange(case[s], device="cuda", dtype=torch.float32) for s in ("frames", "height", "width"))
    t, h, w = (g.reshape(-1) for g in torch.meshgrid(t, h, w, indexing="ij"))
    patches = t.numel()
    if n == 1:
        grid = torch.arange(patches, device="cuda", dtype=torch.float32)[:, None]
    else:
        grid = torch.stack([torch.zeros_like(t), t, h, w][-n:], 1)
    ids = torch.zeros(case["batch"], case["text"] + patches, n, device="cuda")
    ids[:, case["text"]:] = grid
    ids[:, case["text"]:, -2:] += inputs.whole(0, 64, case["batch"], 1, min(n, 2)).float()
    if case["far"]:
        ids[:, case["text"]:, 0] += inputs.whole(0, case["far"], case["batch"], 1).float()
    return ids


def prepare(case, seed):
    kind, inputs = case["kind"], _Inputs(seed)
    state = {"kind": kind, "train": case.get("train", False)}
    if kind == "norm":
        batch, tokens, width, dtype = case["batch"], case["tokens"], case["width"], DTYPES[case["dtype"]]
        # a residual stream: channels of their own mean and spread, a few of them far larger than the rest
        spread = 0.5 + inputs.uniform(width) + 15 * (inputs.uniform(width) < 0.004)
        state["x"] = (inputs.normal(batch, tokens, width, dtype=torch.float32) * spread + inputs.normal(width, std=0.3, dtype=torch.float32)).to(dtype)
        state["plus_one"] = case["weights"] == "modulation"
        state["eps"] = 1e-6
        state["weight"] = state["bias"] = None
        if case["weights"] == "modulation":   # two of the chunks that a modulation projection leaves side by side
            state["bias"], state["weight"], _ = inputs.normal(batch, 1, 3 * width, std=0.2, dtype=dtype).chunk(3, dim=-1)
        elif case["weights"] == "affine":
            state["weight"], state["bias"] = (0.5 + inputs.uniform(width)).to(dtype), inputs.normal(width, std=0.2, dtype=dtype)
        state["wanted"] = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
        if state["train"]:
            state["dy"] = inputs.normal(batch, tokens, width, dtype=dtype)
            for t in state["wanted"]:
                t.requires_grad_(True)
        return state
    if kind in ("rope", "table"):
        state["axes"], state["ids"] = _axes(case), _ids(case, inputs)
        if kind == "table":
            return state
        dim, batch, tokens = sum(state["axes"]), case["batch"], state["ids"].shape[1]
        heads, kv, dtype = case["heads"], case["kv_heads"], DTYPES[case["dtype"]]
        # q and k where a projection of q, k and v leaves them: [batch, tokens, all heads, dim] seen as [batch, heads, tokens, dim]
        fused = inputs.normal(batch, tokens, heads + 2 * kv, dim, dtype=dtype).transpose(1, 2)
        state["q"], state["k"] = fused[:, :heads], fused[:, heads:heads + kv]
        if state["train"]:
            state["q"], state["k"] = state["q"].detach().requires_grad_(True), state["k"].detach().requires_grad_(True)
            state["dq"], state["dk"] = inputs.normal(batch, heads, tokens, dim, dtype=dtype), inputs.normal(batch, kv, tokens, dim, dtype=dtype)
        return state
    requests, rows, k, n, rank, adapters = (case[s] for s in ("requests", "rows", "in", "out", "rank", "adapters"))
    state["x"] = inputs.normal(requests, rows, k) if rows > 1 else inputs.normal(requests, k)
    state["w"] = inputs.normal(n, k, std=k ** -0.5)
    state["b"] = inputs.normal(n, std=0.02)
    state["lora_a"] = inputs.normal(adapters, rank, k, std=k ** -0.5)
    state["lora_b"] = inputs.normal(adapters, n, rank, std=0.5 * rank ** -0.5)
    state["scaling"] = 0.5 + inputs.uniform(adapters)
    # one request in five comes without an adapter (-1); rows of one request lie side by side
    adapter = torch.where(inputs.uniform(requests) < 0.2, -1, inputs.whole(0, adapters, requests))
    if rows == 1 and requests > 64:
        adapter = adapter[torch.sort(inputs.whole(0, requests, requests)).values // 12]
    state["adapter"] = adapter.to(torch.int32)
    state["act"] = case["act"]
    return state


def _norm(state):
    x, w, b = state["x"].float(), state["weight"], state["bias"]
    dtype, width = state["x"].dtype, x.shape[-1]
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + state["eps"])
    h = centred * rstd
    if w is None:
        scale, y = 1.0, h
    else:
        scale = w.float() + 1 if state["plus_one"] else w.float()
        y = h * scale + b.float()
    y = y.to(dtype)
    if not state["train"]:
        return (y,)
    dy = state["dy"].float()
    g = dy * scale
    dx = (rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))).to(dtype)
    if w is None:
        return y, dx
    rows = (1,) if w.dim() == 3 else (0, 1)
    return y, dx, (dy * h).sum(rows).view(w.shape).to(w.dtype), dy.sum(rows).view(b.shape).to(b.dtype)


def _cos_sin(ids, axes):
    """[batch, 1, tokens, pairs], from angles in 64 bits."""
    dims = torch.tensor(axes, device=ids.device)
    axis = torch.repeat_interleave(torch.arange(len(axes), device=ids.device), dims // 2)
    first = torch.cumsum(dims // 2, 0) - dims // 2
    place = torch.arange(axis.numel(), device=ids.device) - first[axis]
    freq = torch.pow(10000.0, -2.0 * place.double() / dims[axis].double())
    angle = (ids.double()[..., axis] * freq).unsqueeze(1)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(x, cos, sin):
    pairs = x.float().unflatten(-1, (-1, 2))
    x0, x1 = pairs[..., 0], pairs[..., 1]
    return torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1).flatten(-2).to(x.dtype)


def _rope(state):
    cos, sin = _cos_sin(state["ids"], state["axes"])
    if state["kind"] == "table":
        return torch.stack((cos, -sin, sin, cos), -1).unflatten(-1, (2, 2))
    out = _rotate(state["q"], cos, sin), _rotate(state["k"], cos, sin)
    if state["train"]:
        out += _rotate(state["dq"], cos, -sin), _rotate(state["dk"], cos, -sin)
    return out


def _lora(state):
    x, a, b = state["x"], state["lora_a"], state["lora_b"]
    adapters, rank, k = a.shape
    n = state["w"].shape[0]
    rows = x.reshape(-1, k).float()
    chosen = state["adapter"].long().repeat_interleave(rows.shape[0] // state["adapter"].numel())
    y = rows @ state["w"].float().T + state["b"].float()
    # every row times every adapter's first factor; all but its own adapter's products are dropped
    low = (rows @ a.float().reshape(adapters * rank, k).T).view(-1, adapters, rank)
    mine = chosen[:, None] == torch.arange(adapters, device=x.device)
    low = torch.where(mine[..., None], low * state["scaling"][:, None], 0.0).view(-1, adapters * rank)
    y = y + low @ b.float().permute(0, 2, 1).reshape(adapters * rank, n)
    if state["act"] == "GELU":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.to(x.dtype).view(*x.shape[:-1], n)


def run(state):
    kind = state["kind"]
    if own:
        import triton_kernels as tk

        if kind == "norm":
            y = tk.layer_norm(state["x"], state["weight"], state["bias"], state["eps"], plus_one=state["plus_one"])
            return (y, *torch.autograd.grad(y, state["wanted"], state["dy"])) if state["train"] else (y,)
        if kind == "rope":
            yq, yk = tk.apply_rope_nd(state["q"], state["k"], state["ids"], state["axes"])
            return (yq, yk, *torch.autograd.grad((yq, yk), (state["q"], state["k"]), (state["dq"], state["dk"]))) if state["train"] else (yq, yk)
        if kind == "table":
            return tk.rope_table(state["ids"], state["axes"])
        return tk.linear_lora(state["x"], state["w"], state["b"], state["lora_a"], state["lora_b"], state["adapter"], state["scaling"], activation=state["act"])
    with torch.no_grad():
        if kind == "norm":
            return _norm(state)
        return _lora(state) if kind == "lora" else _rope(state)


def _tokens(case):
    return case["batch"] * (case["text"] + case["frames"] * case["height"] * case["width"])


def work(case):
    kind = case["kind"]
    size = 4.0 if case.get("dtype") == "fp32" else 2.0
    if kind == "norm":
        values = case["batch"] * case["tokens"] * case["width"]
        weights = {"none": 0, "affine": 2, "modulation": 2 * case["batch"]}[case["weights"]] * case["width"]
        # forward reads x and writes y; the backward pass reads x and dy and writes dx and the weights' gradients
        return {"bytes": size * ((5 if case["train"] else 2) * values + (3 if case["train"] else 1) * weights), "flops": (23.0 if case["train"] else 8.0) * values}
    if kind == "lora":
        m, k, n, r = case["requests"] * case["rows"], case["in"], case["out"], case["rank"]
        used = min(case["adapters"], case["requests"])
        return {"bytes": 2.0 * (m * k + n * k + n + m * n + used * r * (k + n)) + 4.0 * (case["requests"] + case["adapters"]), "flops": 2.0 * m * (n * k + r * (k + n))}
    tokens, dim = _tokens(case), sum(_axes(case))
    ids = 4.0 * tokens * len(_axes(case))
    if kind == "table":
        return {"bytes": ids + 8.0 * tokens * dim, "flops": 20.0 * tokens * dim}
    values = tokens * dim * (case["heads"] + case["kv_heads"])
    passes = 2 if case["train"] else 1
    return {"bytes": passes * (size * 2 * values + ids), "flops": passes * (3.0 * values + 20.0 * tokens * dim)}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "norm":
            x = state["x"].double()
            var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
            h = (x - mean) / torch.sqrt(var + state["eps"])
            w, b = state["weight"], state["bias"]
            gain = torch.ones_like(x[0, 0]) if w is None else w.double() + (1.0 if state["plus_one"] else 0.0)
            y = h * gain + (0.0 if b is None else b.double())
            if not state["train"]:
                return (y,)
            dy = state["dy"].double()
            g = gain * dy
            # the part of g along the row of ones and along h is taken out
            dx = (g - g.sum(-1, keepdim=True) / x.shape[-1] - h * ((h * g).sum(-1, keepdim=True) / x.shape[-1])) / torch.sqrt(var + state["eps"])
            if w is None:
                return y, dx
            by = "bln,bln->bn" if w.dim() == 3 else "bln,bln->n"
            return y, dx, torch.einsum(by, dy, h).reshape(w.shape), torch.einsum(by, dy, torch.ones_like(h)).reshape(b.shape)
        if case["kind"] in ("rope", "table"):
            turns = []
            for i, d in enumerate(state["axes"]):
                for j in range(d // 2):
                    turns.append(state["ids"][..., i].double() / 10000.0 ** (2.0 * j / d))
            phase = torch.stack(turns, -1)
            phase = torch.polar(torch.ones_like(phase), phase)
            if case["kind"] == "table":
                return torch.stack((phase.real, -phase.imag, phase.imag, phase.real), -1).unflatten(-1, (2, 2)).unsqueeze(1)
            phase = phase.unsqueeze(1)

            def turned(x, by):
                return torch.view_as_real(torch.view_as_complex(x.double().contiguous().unflatten(-1, (-1, 2))) * by).flatten(-2)

            out = turned(state["q"], phase), turned(state["k"], phase)
            return out + (turned(state["dq"], phase.conj()), turned(state["dk"], phase.conj())) if state["train"] else out
        x = state["x"].double()
        rows = x.reshape(-1, x.shape[-1])
        y = rows @ state["w"].double().T + state["b"].double()
        owner = state["adapter"].repeat_interleave(rows.shape[0] // state["adapter"].numel())
        for i in owner.unique().tolist():
            if i < 0:
                continue
            at = (owner == i).nonzero()[:, 0]
            y[at] += float(state["scaling"][i]) * ((rows[at] @ state["lora_a"][i].double().T) @ state["lora_b"][i].double().T)
        if state["act"] == "GELU":
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        return y.reshape(*x.shape[:-1], -1)
