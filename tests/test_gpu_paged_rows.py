"""Rows of paged attention that see no key, and values that are not finite, at every head size and in every form of the work:
one part, parts joined by a second launch, parts joined by the wave that arrives last."""
import pytest
import torch

import paged_oracle as po
from common import TINY, QWEN3_NEXT, D128
from test_gpu_paged import BF16, DEV, EVEN, F32, NAN, Batch, attend, contexts  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n,pos", [(TINY, 1, 40), (QWEN3_NEXT, 1, 3000), (D128, 4, 3000), (QWEN3_NEXT, 60, 40), (TINY, 60, 3000),
                                     (QWEN3_NEXT, 600, 900), (D128, 700, 300)], ids=str)
def test_rows_that_see_nothing_are_zero_whatever_their_gate(contexts, s, n, pos, dtype):  # noqa: F811
    """A sequence without pages and the tokens of others outside their table's positions, with gates of NaN and infinities as an
    idle place's rows may hold them: zero, and the other rows as the formula has them."""
    b = Batch(n, s, [pos, pos, pos, 5], n, 32, dtype)
    top = b.table.shape[1] * 32
    b.pos = [pos, pos, top, 5]
    b.table[1] = -1
    junk = torch.tensor([NAN, float("inf"), -float("inf"), NAN]).repeat(s.D // 4)
    b.qg[1:3, :, :, s.D:] = junk
    out = attend(contexts(s), b)
    assert (out[1:3] == 0).all()
    b.new[0] = b.new[3] = min(n, 50)  # (of the others, the first tokens)
    b.check(out)
    # before position 0: the first token of two, or none of one
    if 2 <= n <= 60:
        c = Batch(n, s, [0], n, 32, dtype)
        c.pos = [-1]
        c.qg[:, 0, :, s.D:] = junk
        out = attend(contexts(s), c)
        assert (out[0, 0] == 0).all()
        c.check(out)


# few tokens in one part and in several, chunks joined by a second launch and by the last wave (64 dims: copies and cleaning by half the
# waves each)
@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n,pos", [(TINY, 1, 30), (TINY, 6, 3000), (TINY, 8, 40), (D128, 4, 2000), (D128, 8, 70), (TINY, 9, 70), (TINY, 90, 1000),
                                     (D128, 70, 500), (D128, 9, 3000), (TINY, 4200, 0), (D128, 1100, 1000), (EVEN, 1100, 500)], ids=str)
def test_values_not_finite(contexts, s, n, pos, dtype, bad):  # noqa: F811
    """A value that is not finite, of a token of the chunk or of one before: what sees it is not finite in its dim and keeps its
    other dims; earlier tokens keep their bits. Before a window it changes nothing at all."""
    b = Batch(n, s, [pos, pos // 2], n, 32, dtype, lens=[n, n - n // 3])
    clean = attend(contexts(s), b)
    dim, rest = 3, [i for i in range(s.D) if i != 3]
    pages = b.table[0].tolist()
    for at in {pos + n // 2, pos + n - 1, pos // 2}:
        was = po.rows_of(b.vpool, pages, s.D, b.vi)[at].clone()
        row = was.clone()
        row[:, dim] = bad
        po.put_rows(b.vpool, pages, s.D, b.vi, [at], [row])
        got = attend(contexts(s), b)
        first = max(at - pos, 0)
        assert torch.equal(got[0, :first], clean[0, :first]) and torch.equal(got[1], clean[1])
        assert not got[0, first:, :, dim].isfinite().any()
        # (the other dims' terms are the same, added in the same order or tile by tile)
        err = (got[0, first:, :, rest].double() - clean[0, first:, :, rest].double()).abs()
        assert (err <= 2 * po.HALF[dtype] * clean[0, first:, :, rest].double().abs() + (pos + n) * 2.0 ** -23 * 8).all()
        if at < pos:
            hidden = attend(contexts(s), b, pos - at, 0)
            po.put_rows(b.vpool, pages, s.D, b.vi, [at], [was])
            assert torch.equal(hidden, attend(contexts(s), b, pos - at, 0))
        po.put_rows(b.vpool, pages, s.D, b.vi, [at], [was])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n,pos", [(TINY, 1, 400), (TINY, 3, 400), (D128, 4, 400), (TINY, 70, 400), (D128, 60, 400), (EVEN, 700, 400), (D128, 1100, 200)], ids=str)
def test_hidden_memory_may_hold_anything(contexts, s, n, pos, dtype):  # noqa: F811
    """Keys and values that are not finite before the window and behind the last row, at every head size."""
    window, sinks = 80, 3
    b = Batch(n, s, [pos], n, 32, dtype)
    clean = attend(contexts(s), b, window, sinks)
    assert not clean.isnan().any()
    junk = torch.tensor([NAN, float("inf"), -float("inf"), 65504.0]).repeat(s.D // 4).expand(s.NKV, s.D)
    pages = b.table[0].tolist()
    hidden = list(range(sinks, pos - window + 1)) + list(range(pos + n, len(pages) * 32))
    for pool, place in ((b.kpool, b.ki), (b.vpool, b.vi)):
        po.put_rows(pool, pages, s.D, place, hidden, [junk] * len(hidden))
    assert torch.equal(attend(contexts(s), b, window, sinks), clean)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 4, 60])
def test_tokens_past_the_rope_table(qw, n, dtype):
    """A sequence that reaches the end of the context's rope table, in a table whose columns are held to its positions: appended
    and attended up to the end, zeros from there on, the memory of the wider table's pages as it was; the same by `lens`."""
    s, end, page = TINY, 96, 32
    att = qw.Attention(s.NH, s.NKV, s.D, s.R, s.theta, s.eps, max_ctx=end, max_tokens=64)
    b = Batch(n, s, [end - n // 2, 17], n, page, dtype)  # (of one token the first is past the end)
    wide = torch.cat([b.table, torch.full((2, 3), -1, dtype=torch.int32)], 1)[:, :5]
    kpool, vpool, _, pos = b.dev()
    table = wide.to(DEV)
    k, v = (b.r(2, n, s.NKV, s.D).to(dtype).to(DEV) for _ in "kv")
    qg = b.qg.to(DEV)
    q_out, out = (torch.full((2, n, s.NH, s.D), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    before = kpool.clone(), vpool.clone()
    att.paged_append(k, v, kpool, vpool, table, pos, q=qg[..., :s.D], q_out=q_out)
    att.paged_attend(q_out, kpool, vpool, table[:, :end // page], pos, out, gate=qg[..., s.D:])
    short = torch.full_like(out, 7.0)
    lens = torch.tensor([n // 2, n], dtype=torch.int32, device=DEV)
    att.paged_attend(q_out, kpool, vpool, table, pos, short, gate=qg[..., s.D:], lens=lens)
    torch.cuda.synchronize()
    assert (q_out[0, n // 2:] == 0).all() and (out[0, n // 2:] == 0).all() and (short[0, n // 2:] == 7).all()
    for pool, was in zip((kpool, vpool), before):
        rows, old = (po.rows_of(x.cpu(), b.table[0].tolist(), s.D, b.ki if pool is kpool else b.vi) for x in (pool, was))
        assert torch.equal(rows[end:].view(torch.int16), old[end:].view(torch.int16))
    b.kpool, b.vpool = kpool.cpu(), vpool.cpu()
    b.qg[..., :s.D] = q_out.cpu()
    b.new[0] = n // 2
    b.check(out)
    b.check(short, left=7)
    att.close()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n,pos", [(QWEN3_NEXT, 1, 700), (D128, 5, 900), (TINY, 60, 300), (QWEN3_NEXT, 700, 100)], ids=str)
def test_a_query_that_is_not_finite_stays_in_its_row(contexts, s, n, pos, dtype):  # noqa: F811
    """A NaN or an infinity in one head's query of one token, and in one element of a gate: the other rows keep their bits."""
    b = Batch(n, s, [pos], n, 32, dtype)
    clean = attend(contexts(s), b)
    t, h = n // 2, s.NH - 1
    for x in (NAN, float("inf")):
        b.qg[0, t, h, 5] = x
        got = attend(contexts(s), b)
        assert got[0, t, h].isnan().all()
        got[0, t, h] = clean[0, t, h]
        assert torch.equal(got, clean)
    b = Batch(n, s, [pos], n, 32, dtype)
    b.qg[0, t, h, s.D + 5] = NAN
    got = attend(contexts(s), b)
    assert got[0, t, h, 5].isnan()
    got[0, t, h, 5] = clean[0, t, h, 5]
    assert torch.equal(got, clean)
