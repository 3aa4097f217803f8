"""Paged attention where its work is split and joined: long sequences, batches of many sequences, row counts at the border of
its forms, values that are not finite in split sequences, and one workspace for calls of both forms. Long cases are held
against the 64-bit oracle at tokens spread over the chunk."""
import pytest
import torch

import paged_oracle as po
from common import TINY, QWEN3_NEXT, D128, Shape
from test_gpu_paged import (BF16, DEV, EVEN, F32, MANY, NAN, Batch, attend, check_append, contexts,  # noqa: F401 (a fixture)
                            rope_table)

pytestmark = pytest.mark.gpu


def check_tokens(b, out, tokens, window=0, sinks=0, sequences=None):
    """out [n_seq, n, heads, d] at `tokens` of every sequence (of `sequences`) against the oracle."""
    d = b.s.D
    out = out.double().cpu()
    for i in range(len(b.pos)) if sequences is None else sequences:
        pages = b.table[i].tolist()
        keys, values = po.rows_of(b.kpool, pages, d, b.ki), po.rows_of(b.vpool, pages, d, b.vi)
        there = torch.ones(len(keys), dtype=torch.bool)
        for t in sorted({x for x in tokens if 0 <= x < b.new[i]}):
            q = b.qg[i, t:t + 1]
            want, bound = po.attend(q[..., :d], keys, values, there, b.pos[i] + t, window, sinks, d ** -0.5, q[..., d:], b.dtype)
            err = (out[i, t] - want[0]).abs()
            assert (err <= bound[0]).all(), f"sequence {i}, token {t}: {float(err.max()):.3e} off, bound {float(bound.max()):.3e}"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,n", [(EVEN, 16), (EVEN, 17), (EVEN, 32), (EVEN, 33), (MANY, 8), (MANY, 9), (QWEN3_NEXT, 5)], ids=str)
def test_row_counts_at_the_border_of_the_forms(contexts, s, n, dtype):  # noqa: F811
    b = Batch(n, s, [150, 3], n, 32, dtype, lens=[n, n - 1])
    b.check(attend(contexts(s), b), left=7)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 20])
@pytest.mark.parametrize("nh,nkv,d", [(32, 1, 64), (32, 2, 256), (16, 8, 128), (32, 32, 64)])
def test_head_groups(qw, nh, nkv, d, n, dtype):
    """Groups of 32, 16, 2 and 1 query heads to a KV head: a token's rows fill a tile, several or a part of one."""
    s = Shape(nh, nkv, d, 0)
    att = qw.Attention(nh, nkv, d, 0, max_ctx=64, max_tokens=8)
    b = Batch(nh + n, s, [70, 0, 33], n, 32, dtype, lens=[n, 1, n - 1])
    b.check(attend(att, b), left=7)
    b.check(attend(att, b, 20, 2), 20, 2, left=7)
    att.close()


@pytest.mark.parametrize("s,pos,n,page,dtype,window,sinks", [
    (TINY, [20000], 1, 64, F32, 0, 0), (TINY, [20000, 40, 9000], 3, 32, BF16, 0, 0), (QWEN3_NEXT, [9000], 4, 256, F32, 0, 0),
    (D128, [12000, 31], 1, 64, BF16, 8000, 200),
    # few items, cut in many parts; few items in parts of more than 64 blocks
    (TINY, [20000], 61, 64, F32, 0, 0), (EVEN, [34000], 512, 128, BF16, 0, 0), (TINY, [17000], 2100, 64, BF16, 0, 0),
    # many items, in runs of more than 64 blocks; the same past a window
    (TINY, [14000], 4200, 64, BF16, 0, 0), (TINY, [12000], 4200, 64, F32, 9000, 100)], ids=str)
def test_long_sequences(contexts, s, pos, n, page, dtype, window, sinks):  # noqa: F811
    b = Batch(n + window, s, pos, n, page, dtype)
    out = attend(contexts(s), b, window, sinks)
    assert not out.isnan().any()
    check_tokens(b, out, {0, 1, n // 3, n // 2, n - 2, n - 1} | set(range(0, n, max(1, n // 24))), window, sinks)


@pytest.mark.parametrize("count,n,dtype", [(64, 1, F32), (65, 1, BF16), (300, 2, F32), (300, 40, BF16), (1100, 33, F32), (1500, 1, BF16)])
def test_batches_of_many_sequences(contexts, count, n, dtype):  # noqa: F811
    pos = [(37 * i) % 97 for i in range(count)]
    lens = [n if i % 3 == 0 else i % (n + 1) for i in range(count)]  # none among them
    b = Batch(count, TINY, pos, n, 32, dtype, lens=lens)
    out = attend(contexts(TINY), b)
    for i, m in enumerate(b.new):
        assert not out[i, :m].isnan().any() and (out[i, m:] == 7).all()
    check_tokens(b, out, {0, n // 2, n - 1}, sequences=range(0, count, 1 + count // 60))


@pytest.mark.parametrize("bad", [NAN, float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("n,dtype", [(4, F32), (4, BF16), (60, F32), (60, BF16), (300, F32), (700, BF16), (1100, F32), (2100, BF16)])
def test_values_not_finite_in_split_sequences(contexts, n, dtype, bad):  # noqa: F811
    """A value that is not finite reaches the tokens that see it, in its dim, and leaves the earlier tokens' bits alone."""
    s, pos, dim = QWEN3_NEXT, 3000, 5
    b = Batch(n, s, [pos], n, 64, dtype)
    clean = attend(contexts(s), b)
    check_tokens(b, clean, {0, n // 2, n - 1})
    at = pos + n // 2
    pages = b.table[0].tolist()
    row = po.rows_of(b.vpool, pages, s.D, b.vi)[at]
    row[:, dim] = bad
    po.put_rows(b.vpool, pages, s.D, b.vi, [at], [row])
    got = attend(contexts(s), b)
    assert torch.equal(got[:, :n // 2], clean[:, :n // 2])
    assert not got[:, n // 2:, :, dim].isfinite().any()
    rest = [i for i in range(s.D) if i != dim]
    err = (got[:, n // 2:, :, rest].double() - clean[:, n // 2:, :, rest].double()).abs()
    # (sums that are not finite in one dim leave the others' terms as they are, in the same order or tile by tile)
    assert (err <= 2 * po.HALF[dtype] * clean[:, n // 2:, :, rest].double().abs() + (pos + n) * 2.0 ** -23 * 8).all()


def test_one_workspace_for_both_forms(contexts):  # noqa: F811
    """Calls of both forms one after the other in one workspace, eager and as one captured graph replayed between them."""
    s = QWEN3_NEXT
    att = contexts(s)
    ws = torch.full((att.paged_workspace(),), 0xA5, dtype=torch.uint8, device=DEV)
    calls = []
    for n, pos, dtype in ((1, [700, 90], F32), (40, [500, 20], BF16), (3, [64, 900], BF16), (300, [33, 300], F32)):
        b = Batch(n, s, pos, n, 64, dtype)
        kpool, vpool, table, at = b.dev()
        qg, want = b.qg.to(DEV), attend(att, b)
        out = torch.empty_like(want)
        calls.append((want, out, lambda qg=qg, k=kpool, v=vpool, t=table, p=at, o=out: att.paged_attend(
            qg[..., :s.D], k, v, t, p, o, gate=qg[..., s.D:], workspace=ws)))
    def run_all():
        for _, _, call in calls:
            call()
    def check_all():
        torch.cuda.synchronize()
        for want, out, _ in calls:
            assert torch.equal(out, want)
            out.fill_(NAN)
    for _ in range(3):
        run_all()
        check_all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run_all()
    for _ in range(3):
        g.replay()
        check_all()
        run_all()
        check_all()


@pytest.mark.parametrize("n", [1, 4, 30, 400])
def test_a_captured_call_follows_lengths_and_tables(contexts, n):  # noqa: F811
    """A captured call replayed as positions, lengths and the order of sequences change on the device: as the eager call."""
    s = QWEN3_NEXT
    att = contexts(s)
    b = Batch(n, s, [2000, 1500, 900], n, 64, BF16, lens=[n, n, n])
    kpool, vpool, table, pos = b.dev()
    qg = b.qg.to(DEV)
    ws = torch.empty(att.paged_workspace(), dtype=torch.uint8, device=DEV)
    out = torch.full((3, n, s.NH, s.D), 7.0, dtype=BF16, device=DEV)
    call = lambda o, w: att.paged_attend(qg[..., :s.D], kpool, vpool, table, pos, o, gate=qg[..., s.D:], lens=b.lens, workspace=w)  # noqa: E731
    call(out, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out, ws)
    for at, new, order in (([2000, 1500, 900], [n] * 3, [0, 1, 2]), ([3, 1500, 0], [n, 1, n], [0, 1, 2]), ([900, 2000, 33], [0, n, 1], [2, 0, 1]),
                           ([1999, 70, 899], [1, n, 0], [0, 1, 2])):
        pos.copy_(torch.tensor(at)), b.lens.copy_(torch.tensor(new)), table.copy_(b.table[order])
        out.fill_(7.0)
        want = out.clone()
        g.replay()
        call(want, None)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        b2 = Batch(n, s, [2000, 1500, 900], n, 64, BF16, lens=[n, n, n])
        b2.pos, b2.new, b2.table = at, new, b.table[order]
        check_tokens(b2, out, {0, n - 1})


@pytest.mark.parametrize("s,n,lens,dtype", [(EVEN, 1100, [1100, 987, 0], F32), (QWEN3_NEXT, 650, [650, 1, 649], BF16), (MANY, 420, None, F32),
                                            (Shape(4, 4, 128, 64), 1400, [1400, 1399, 5], BF16)], ids=str)
def test_append_many_rows(contexts, s, n, lens, dtype):  # noqa: F811
    """Chunks of so many rows that a half-wave takes several heads, head counts that do not divide among them too."""
    b = Batch(n, s, [31, 0, 77], n, 64, dtype, lens=lens)
    k, v, qn, kn = b.r(3, n, s.NKV, s.D).to(dtype), b.r(3, n, s.NKV, s.D).to(dtype), b.r(s.D, sd=0.2), b.r(s.D, sd=0.2)
    rope = rope_table(s, 2048)
    check_append(contexts(s), b, k, v, qn, kn, rope)
    check_append(contexts(s), b, k, v, None, kn, rope, with_q=False)


@pytest.mark.parametrize("n", [1, 4, 90])
def test_sequences_share_a_prompts_pages(contexts, n):  # noqa: F811
    """Three sequences whose first pages are one and the same, two of them all but their last page."""
    b = Batch(n, QWEN3_NEXT, [500, 500, 300], n, 32, F32)
    b.table[1, :15], b.table[2, :9] = b.table[0, :15], b.table[0, :9]
    b.check(attend(contexts(QWEN3_NEXT), b))
