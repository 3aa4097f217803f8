"""The paged-attention operators in 64 bits, token by token, with worst-case rounding bounds of the kernels' arithmetic:
the oracle of test_gpu_paged.py. Pools are looked at position by position through the cache's block layout."""
import math

import torch

EPS32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def block_places(d):
    """Element of a 32-position block that holds (position kb, dim) of K and of V: [32, d] each."""
    k = torch.empty(32, d, dtype=torch.long)
    v = torch.empty(32, d, dtype=torch.long)
    for kb in range(32):
        for e in range(d):
            k[kb, e] = ((((e // 32) * 2 + (kb // 4) % 2) * 4 + (e // 8) % 4) * 16 + (kb // 8) * 4 + kb % 4) * 8 + e % 8
            v[kb, e] = (((e // 16) * 4 + kb // 8) * 16 + e % 16) * 8 + kb % 8
    return k, v


def rows_of(pool, pages, d, place):
    """[positions, KV heads, d] of a sequence's pages (CPU tensors); pages outside the pool read as NaN."""
    n_pages, nkv, per = pool.shape
    out = torch.full((len(pages), per // (32 * d), 32, nkv, d), float("nan"), dtype=pool.dtype)
    for i, p in enumerate(pages):
        if 0 <= p < n_pages:
            out[i] = pool[p].view(nkv, -1, 32 * d)[..., place].permute(1, 2, 0, 3)
    return out.flatten(0, 2)


def put_rows(pool, pages, d, place, at, rows):
    """Writes rows [n, KV heads, d] at positions `at` of a sequence's pages; positions without a page are left out."""
    n_pages, nkv, per = pool.shape
    page = per // d
    flat = pool.view(n_pages, nkv, page // 32, 32 * d)
    for p, r in zip(at, rows):
        if 0 <= p < len(pages) * page and 0 <= pages[p // page] < n_pages:
            flat[pages[p // page], :, p % page // 32][:, place[p % 32]] = r.to(pool.dtype)


def turned(x, w, rope, positions, eps):
    """(norm and rotation of x [n, heads, d] at `positions`, a bound on the fp32 arithmetic's error of each element)"""
    x = x.double()
    d, r = x.shape[-1], 2 * rope.shape[1]
    y = x
    if w is not None:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + w.double())
    cos, sin = rope.double()[positions].unbind(-1)
    cos, sin = cos[:, None], sin[:, None]
    lo, hi = y[..., :r // 2], y[..., r // 2:r]
    out = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, y[..., r:]], -1)
    mag = torch.cat([(lo * cos).abs() + (hi * sin).abs(), (hi * cos).abs() + (lo * sin).abs(), y[..., r:].abs()], -1)
    # half the relative error of a sum of d squares (d / 32 in a lane, five joins, a rounding a square), the mean, the
    # root, its reciprocal, two products, 1 + w; the rotation's two products and sum
    rel = (d / 32 + 5 + 2) / 2 + 6 + 2
    return out, rel * EPS32 * mag


def attend(q, krows, vrows, there, pos, window, sinks, scale, gate, dtype):
    """One sequence: q [n, heads, d], krows and vrows [positions, KV heads, d], there [positions] (a key has a page).
    Returns (out, bound) [n, heads, d] in 64 bits."""
    n, nh, d = q.shape
    nkv = krows.shape[1]
    out, bound = torch.zeros(n, nh, d, dtype=torch.float64), torch.zeros(n, nh, d, dtype=torch.float64)
    j = torch.arange(krows.shape[0])
    for t in range(n):
        p = pos + t
        if not 0 <= p < krows.shape[0]:
            continue
        sees = (j <= p) & there
        if window:
            sees &= (j > p - window) | (j < sinks)
        if not sees.any():
            continue
        for h in range(nh):
            k, v = krows[sees, h // (nh // nkv)].double(), vrows[sees, h // (nh // nkv)].double()
            x = q[t, h].double()
            s = scale * (k @ x)
            w = torch.softmax(s, 0)
            o = w @ v
            wv = w @ v.abs()
            keys = len(s)
            # a score: every product exact but for the query's parts (2^-21 of its largest in fp32 rows, where 22 bits are
            # kept; nothing in bf16 rows), a sum of d, the scale and the maximum's subtraction; as matrix instructions may
            # truncate where others round, sums count double
            mag = scale * float((k.abs() @ x.abs()).max())
            ds = mag * (2 * d + 8) * EPS32 + scale * float(x.abs().max()) * float(k.abs().sum(-1).max()) * 2.0 ** -21
            ds = ds + 2 * EPS32 * float(s.abs().max())
            # a weight: its exponential of 2 units; one fp16 part in bf16 rows, 21 bits in fp32 rows
            dw = ds + 4 * EPS32 + (2.0 ** -11 if dtype is torch.bfloat16 else 2.0 ** -21)
            # numerator and denominator are off by dw each; their sums; weights below fp16's normal range (2^-21 of the
            # largest with the kernels' shift, to 2^-31 absolutely)
            e = 2 * dw * wv + 2 * (keys + 16) * EPS32 * wv + keys * 2.0 ** -31 * v.abs().amax(0) / float(torch.exp(s - s.max()).sum())
            if gate is not None:
                g = 1 / (1 + torch.exp(-gate[t, h].double()))
                o = o * g
                e = e * g + o.abs() * (8 + 2 * gate[t, h].double().abs()) * EPS32
            out[t, h], bound[t, h] = o, 1.01 * (e + HALF[dtype] * (o.abs() + e)) + 1e-37
    return out, bound
