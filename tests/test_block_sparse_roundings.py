"""Attention over listed blocks against float64 with a bound of the roundings that it has and no others: probabilities and result in bf16, the sum of the rounded
probabilities, everything else fp32. q and the scale are not rounded."""
import math

import pytest
import torch

import triton_kernels as tk
from util import DEV, randn, seeded

HALF = torch.finfo(torch.bfloat16).eps / 2
SHAPES = [(2, 1, 300, 1000, 128, 9, 1.0, None), (2, 2, 200, 640, 64, 10, 4.0, None), (4, 1, 130, 3000, 128, 30, 4.0, None), (2, 2, 256, 640, 128, 5, 2.0, 0.3), (3, 1, 1, 4000, 128, 40, 4.0, None),
          (2, 1, 140, 900, 64, 14, 1.0, -0.7)]


def inputs(Hq, Hk, Lq, Lk, D, count, std):
    g = seeded(Lq + Lk + D)
    q, k, v = randn(g, 1, Hq, Lq, D, dtype=torch.bfloat16, std=std), randn(g, 1, Hk, Lk, D, dtype=torch.bfloat16), randn(g, 1, Hk, Lk, D, dtype=torch.bfloat16)
    have = -(-Lk // 64)
    blocks = torch.stack([torch.randperm(have, generator=g)[:count] for _ in range(Hq * -(-Lq // 128))]).view(1, Hq, -1, min(count, have)).to(torch.int32)
    return q, k, v, blocks


def rows(q, k, v, blocks):
    """Each (head, block of queries): its queries, listed keys and values in float64, and where it stands."""
    per = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        for t in range(blocks.shape[2]):
            tokens = torch.cat([torch.arange(j * 64, min(j * 64 + 64, k.shape[2])) for j in blocks[0, h, t].tolist()])
            at = slice(t * 128, min(t * 128 + 128, q.shape[2]))
            yield h, at, q[0, h, at].double(), k[0, h // per, tokens].double(), v[0, h // per, tokens].double()


def expected(q, k, v, blocks, scale):
    """The result, how far a value may be from it, and the root mean square that independent roundings leave.

    With probabilities p (1 + e), the numerator and the sum from the same ones, the result moves by sum p e (v - o) / sum p (1 + e). |e| is half a step, what the
    scores' fp32 sums of D products leave (2^-23 each, of sum |q k| times the scale), the exponent's argument in fp32 (2^-23 of twice the largest score, in base 2) and 2^-21 of the
    exponential; sums over n tokens add 2^-23 each, and the result's own rounding is half a step. Half steps are spread evenly: a third of their square in the mean, at most."""
    D = q.shape[3]
    scale = D ** -0.5 if scale is None else scale
    out, off, mean = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    for h, at, qt, kt, vt in rows(q, k, v, blocks):
        s = qt @ kt.T * scale
        p = torch.softmax(s, -1)
        o = p @ vt
        away = torch.stack([(p[i, :, None] * (vt - o[i]).abs()).sum(0) for i in range(len(o))])
        square = torch.stack([(p[i, :, None] ** 2 * (vt - o[i]) ** 2).sum(0) for i in range(len(o))])
        sums = D * 2.0 ** -23 * (qt.abs() @ kt.abs().T).amax(-1, keepdim=True) * abs(scale) + 2.0 ** -22 * s.abs().amax(-1, keepdim=True) * math.log2(math.e) + 2.0 ** -21
        e = HALF + 1.01 * sums
        err = e / (1 - e) * away + (len(kt) + 64) * 2.0 ** -23 * (p @ vt.abs() + o.abs())
        out[0, h, at], off[0, h, at] = o, err + HALF * (o.abs() + err)
        mean[0, h, at] = ((square + o ** 2) * HALF ** 2 / 3).sqrt()
    return out, off, mean


def beyond(got, want, off, mean):
    """How often a value is beyond its bound, and the root mean square of the differences in parts of what it may be."""
    err = (got.double() - want).abs()
    return int((err > off).sum()), float(err.pow(2).mean().sqrt() / mean.pow(2).mean().sqrt())


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk,Lq,Lk,D,count,std,scale", SHAPES)
def test_roundings(Hq, Hk, Lq, Lk, D, count, std, scale):
    q, k, v, blocks = inputs(Hq, Hk, Lq, Lk, D, count, std)
    got = tk.block_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks.to(DEV), scale).cpu()
    outside, of_mean = beyond(got, *expected(q, k, v, blocks, scale))
    assert outside == 0 and of_mean <= 1.0


@pytest.mark.parametrize("Hq,Hk,Lq,Lk,D,count,std,scale", SHAPES)
def test_the_bound_tells_another_rounding(Hq, Hk, Lq, Lk, D, count, std, scale):
    """On the CPU: the same roundings stay within, q times the scale rounded to bf16 does not where scores are large."""
    q, k, v, blocks = inputs(Hq, Hk, Lq, Lk, D, count, std)
    factor = (D ** -0.5 if scale is None else scale) * math.log2(math.e)
    bound = expected(q, k, v, blocks, scale)
    for rounded in (False, True):
        got = torch.zeros(q.shape, dtype=torch.bfloat16)
        for h, at, qt, kt, vt in rows(q, k, v, blocks):
            s = (qt * factor).bfloat16().double() @ kt.T if rounded else qt @ kt.T * factor
            p = torch.exp2(s - s.amax(-1, keepdim=True)).bfloat16().double()
            got[0, h, at] = (p @ vt / p.sum(-1, keepdim=True)).bfloat16()
        outside, of_mean = beyond(got, *bound)
        if not rounded:
            assert outside == 0 and of_mean <= 1.0
        elif std * abs(factor) * D ** 0.5 >= 4.0 and Hq * Lq >= 100:   # (a few rows are too few roundings of q for their mean to say anything)
            assert of_mean > 1.0
