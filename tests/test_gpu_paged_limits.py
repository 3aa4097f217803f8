"""Paged calls at the ends of their ranges: tables of 2^26 positions, 65,535 sequences. Queries of zero give every key that a
row sees the same weight, so that an output is the mean of those values."""
import pytest
import torch

import paged_oracle as po
from common import Shape
from test_gpu_paged import BF16, DEV, F16, F32

pytestmark = pytest.mark.gpu

S = Shape(4, 1, 64, 0)  # no rotation: positions need no rope table


@pytest.fixture(scope="module")
def att(qw):
    a = qw.Attention(S.NH, S.NKV, S.D, 0, max_ctx=64, max_tokens=8)
    yield a
    a.close()


def pool_of(rows, place, page):
    """[pages, 1, page * D] on the GPU from rows [pages * page, D]"""
    out = torch.empty(len(rows) // page, 1, page // 32, 32 * S.D, dtype=F16, device=DEV)
    out[..., place.flatten().to(DEV)] = rows.view(-1, page // 32, 32 * S.D).unsqueeze(1)
    return out.flatten(2)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 8, 60])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1 << 22, 100)])
def test_the_longest_table(att, n, dtype, window, sinks):
    """A sequence that ends at position 2^26 - 1, its last tokens appended; pages of 65536 positions, four of them over and over but for
    the last."""
    page, pages, d = 65536, 1024, S.D
    top = page * pages
    ki, vi = po.block_places(d)
    g = torch.Generator(device=DEV).manual_seed(n)
    values = torch.randint(0, 4, (5 * page, d), generator=g, device=DEV).to(F16)
    kpool, vpool = pool_of(torch.randn(5 * page, d, generator=g, device=DEV).to(F16), ki, page), pool_of(values, vi, page)
    table = (torch.arange(pages) % 4).to(torch.int32)
    table[-1] = 4
    table = table.to(DEV)[None]
    pos = torch.tensor([top - n], dtype=torch.int32, device=DEV)
    k, v = torch.randn(1, n, 1, d, generator=g, device=DEV).to(dtype), torch.randint(0, 4, (1, n, 1, d), generator=g, device=DEV).to(dtype)
    q = torch.zeros(1, n, S.NH, d, dtype=dtype, device=DEV)
    q_out, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    was = vpool.clone()
    att.paged_append(k, v, kpool, vpool, table, pos, q=q, q_out=q_out)
    att.paged_attend(q_out, kpool, vpool, table, pos, out, window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert (q_out == 0).all()
    values[-n:] = v[0, :, 0].to(F16)
    assert torch.equal(vpool, pool_of(values, vi, page)) and torch.equal(vpool[:4], was[:4])
    sums = torch.cat([torch.zeros(1, d, dtype=torch.float64, device=DEV), values.double().cumsum(0)])
    whole = [sums[(i + 1) * page] - sums[i * page] for i in range(4)]

    def upto(p):  # the sum of positions [0, p)
        i, r = (pages - 1, page) if p == top else divmod(p, page)
        at = 4 if i == pages - 1 else i % 4
        return (i // 4) * sum(whole) + sum(whole[:i % 4], torch.zeros_like(sums[0])) + sums[at * page + r] - sums[at * page]

    for t in range(n):
        p = top - n + t
        first = max(p - window + 1, 0) if window else 0
        kept = min(sinks, first)
        want = (upto(p + 1) - upto(first) + upto(kept)) / (p + 1 - first + kept)
        # weights and weighted values are multiples of 2^8 and add up exactly below 2^32; all of them are at most 2^36, which the
        # joins of at most 512 parts of four waves pass in fewer than 2^10 steps that round
        bound = (2.0 ** 10 * po.EPS32 + po.HALF[dtype]) * want
        err = (out[0, t].double() - want).abs()
        assert (err <= bound).all(), f"token {t}: {float((err / want).max()):.2e}"


@pytest.mark.parametrize("count,n,dtype", [(65535, 1, F32), (65535, 1, BF16), (40000, 8, BF16), (12000, 33, BF16), (5000, 40, F32)])
def test_the_most_sequences(att, count, n, dtype):
    """Each sequence has one page or two of a small pool, in an order of its own, and a length of its own, none among them."""
    page, d, held = 64, S.D, 61
    ki, vi = po.block_places(d)
    g = torch.Generator(device=DEV).manual_seed(count)
    values = torch.randint(0, 4, (held * page, d), generator=g, device=DEV).to(F16)
    kpool, vpool = pool_of(torch.randn(held * page, d, generator=g, device=DEV).to(F16), ki, page), pool_of(values, vi, page)
    i = torch.arange(count, device=DEV)
    table = torch.stack([i % held, (7 * i + 3) % held], 1).to(torch.int32)
    pos, lens = (11 * i % (2 * page - n + 1)).to(torch.int32), (i % (n + 2)).to(torch.int32).clamp(max=n)
    out = torch.full((count, n, S.NH, d), 7.0, dtype=dtype, device=DEV)
    att.paged_attend(torch.zeros_like(out), kpool, vpool, table, pos, out, lens=lens)
    sums = torch.cat([torch.zeros(1, d, dtype=torch.float64, device=DEV), values.double().cumsum(0)])
    for t in range(n):
        end = pos.long() + t + 1
        a, b = table.long().unbind(1)
        one, two = end.clamp(max=page), (end - page).clamp(min=0)
        want = (sums[a * page + one] - sums[a * page] + sums[b * page + two] - sums[b * page]) / end[:, None]
        there = t < lens
        err = (out[:, t].double() - want[:, None]).abs()
        # (whole numbers below 2^24 add up exactly; the reciprocal and the product round)
        bad = err > ((3 * po.EPS32 + po.HALF[dtype] * (1 + 3 * po.EPS32)) * want)[:, None]
        assert not bad[there].any(), f"token {t}: {int(bad[there].sum())} outputs off, first of sequence {int(i[there][bad[there].flatten(1).any(1)][0])}"
        assert (out[~there, t] == 7).all()


def test_append_of_the_most_sequences(att):
    """One token to each of 65,535 sequences at positions of their own, every other page missing."""
    count, page, d = 65535, 32, S.D
    ki, vi = po.block_places(d)
    i = torch.arange(count, device=DEV)
    table = torch.where(i % 2 == 0, i // 2, -1 - i).to(torch.int32)[:, None]
    pool = torch.full(((count + 1) // 2, 1, page * d), 9.0, dtype=F16, device=DEV)
    kpool, vpool = pool.clone(), pool.clone()
    pos = (5 * i % 40).to(torch.int32)  # (some past the page)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(count, 1, 1, d, generator=g, device=DEV) for _ in "kv")
    att.paged_append(k, v, kpool, vpool, table, pos)
    for got, rows, place in ((kpool, k, ki), (vpool, v, vi)):
        want = pool.clone()
        at = ((i % 2 == 0) & (pos < page)).nonzero()[:, 0]
        want[table[at, 0].long()[:, None], 0, place.to(DEV)[pos[at].long()]] = rows[at, 0, 0].to(F16)
        assert torch.equal(got, want)
