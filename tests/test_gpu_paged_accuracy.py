"""Accuracy of paged attention beyond the worst-case bounds of test_gpu_paged.py: outputs whose terms cancel, and the 2-norm of
bf16 outputs' distance from the rounded 64-bit ones. Weights, their sums and the outputs before their one rounding are of fp32
accuracy for rows of either type."""
import math

import pytest
import torch

import paged_oracle as po
from common import TINY, QWEN3_NEXT, D128
from test_gpu_paged import BF16, F16, F32, Batch, attend, contexts  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def half_step(x, dtype):
    """Half the distance between neighbouring numbers of `dtype` around each x (in 64 bits)."""
    _, exponent = torch.frexp(x.abs().clamp(min=2.0 ** -100))
    return torch.ldexp(torch.full_like(x, po.HALF[dtype]), exponent - 1)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n", [(TINY, 1), (TINY, 8), (TINY, 60), (D128, 1), (D128, 8), (D128, 100), (QWEN3_NEXT, 1), (QWEN3_NEXT, 4),
                                 (QWEN3_NEXT, 60)], ids=str)
def test_terms_that_cancel(contexts, s, n, dtype):  # noqa: F811
    """Eight keys whose weighted values sum to about 2^-12 of themselves, in every dim: an error of a weight that a sum of
    ordinary terms hides stands beside the output's own step here.

    The eight are sinks, the pages of the tokens' own positions are missing; every query is a unit vector, so that a score is one
    product, exact, and the bound is small: the exponent's two roundings and that of the scale, an exponential of 2 units, weights in two
    fp16 parts (2^-22), and sums of eight that count double."""
    keys, d, pos = 8, s.D, 64
    b = Batch(n, s, [pos], n, 32, dtype)
    b.table[0, pos // 32:] = -1
    b.qg[..., :d] = 0
    b.qg[..., 0] = 1
    k = torch.zeros(keys, s.NKV, d)
    k[:, :, 0] = b.r(keys, s.NKV)
    k[-1, :, 0] = k[:, :, 0].amax(0)
    k = k.to(F16).double()
    w = torch.softmax(k[:, :, :1], 0)  # [keys, KV heads, 1]: the scale is 1
    v = b.r(keys, s.NKV, d).to(F16).double()
    v[-1] = (-(w[:-1] * v[:-1]).sum(0) / w[-1]).to(F16).double()
    pages = b.table[0].tolist()
    po.put_rows(b.kpool, pages, d, b.ki, range(keys), k)
    po.put_rows(b.vpool, pages, d, b.vi, range(keys), v)
    o, wv = (w * v).sum(0), (w * v.abs()).sum(0)
    assert float((o.abs() / wv).max()) < 2.0 ** -11
    dw = (4 * float(k.abs().max()) + 12) * po.EPS32 + 2.0 ** -22
    e = (dw + 2 * (keys + 16) * po.EPS32) * (wv + o.abs())
    bound = 1.01 * (e + half_step(o.abs() + e, dtype))
    out = attend(contexts(s), b, window=1, sinks=keys, gated=False, scale=1.0).double().cpu()[0]
    err = (out.unflatten(1, (s.NKV, s.G)) - o[:, None]).abs()
    worst = (err / bound[:, None]).max()
    assert worst <= 1, f"{float(worst):.2f} times the bound; {float((err > bound[:, None]).double().mean()):.2%} of the outputs are off"


@pytest.mark.parametrize("s,pos,n", [(QWEN3_NEXT, 700, 1), (QWEN3_NEXT, 300, 4), (QWEN3_NEXT, 200, 40), (D128, 500, 8), (D128, 100, 90),
                                     (TINY, 900, 2), (TINY, 50, 100)], ids=str)
def test_bf16_outputs_are_the_rounded_ones_but_at_borders(contexts, s, pos, n):  # noqa: F811
    """An error of 2^-20 of an output before its rounding (16 units of fp32) moves the rounded one by a step, 2^-7 of it at most,
    where a border lies within the error: the 2-norm of the difference from rounded 64-bit outputs is sqrt(2^-20 2^-7) of
    theirs at most, 8.6e-5. Weights of 11 bits make it 9e-4."""
    b = Batch(n + pos, s, [pos], n, 32, BF16)
    want = b.want()[0][0].to(BF16).double()
    got = attend(contexts(s), b).double().cpu()[0]
    far = float((got - want).norm() / want.norm())
    assert far <= math.sqrt(2.0 ** -27), f"{far:.2e}"
