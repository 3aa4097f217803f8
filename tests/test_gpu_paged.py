"""Attention of batches over a paged K/V cache on the GPU: appending (norm, rotation, pages) and attending (decode, verify,
chunks; windows and sinks) against the 64-bit restatements of paged_oracle.py, and a run of both as a serving loop makes it."""
import math

import pytest
import torch

import paged_oracle as po
from common import TINY, TINY_GGUF, QWEN3_NEXT, D128, Shape

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MANY, EVEN = Shape(32, 8, 128, 128), Shape(8, 8, 64, 64)
NAN = float("nan")


@pytest.fixture(scope="module")
def contexts(qw):
    made = {}

    def get(s):
        if repr(s) not in made:
            made[repr(s)] = qw.Attention(s.NH, s.NKV, s.D, s.R, s.theta, s.eps, max_ctx=2048, max_tokens=64)
        return made[repr(s)]

    yield get
    for a in made.values():
        a.close()


class Batch:
    """Seeded pools, page tables and rows of a batch: pages in random order, everything that no sequence owns NaN."""

    def __init__(self, seed, s, pos, n, page, dtype, lens=None, spare=2, keys_sd=1.0):
        self.s, self.pos, self.n, self.page, self.dtype = s, pos, n, page, dtype
        self.new = [min(max(x, 0), n) for x in lens] if lens is not None else [n] * len(pos)
        g = torch.Generator().manual_seed(seed)
        self.r = r = lambda *shape, sd=1.0: torch.randn(shape, generator=g) * sd
        b = len(pos)
        pages = max(1, max(-(-(max(p, 0) + n) // page) for p in pos))
        total = b * pages + spare
        self.table = torch.randperm(total, generator=g)[:b * pages].view(b, pages).to(torch.int32)
        self.kpool = torch.full((total, s.NKV, page * s.D), NAN, dtype=F16)
        self.vpool = self.kpool.clone()
        self.ki, self.vi = po.block_places(s.D)
        for i in range(b):
            keys = max(0, pos[i] + self.new[i])
            po.put_rows(self.kpool, self.table[i].tolist(), s.D, self.ki, range(keys), r(keys, s.NKV, s.D, sd=keys_sd))
            po.put_rows(self.vpool, self.table[i].tolist(), s.D, self.vi, range(keys), r(keys, s.NKV, s.D))
        self.qg = r(b, n, s.NH, 2 * s.D).to(dtype)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens is not None else None

    def dev(self):
        """(kpool, vpool, table, pos) on the GPU"""
        return self.kpool.to(DEV), self.vpool.to(DEV), self.table.to(DEV), torch.tensor(self.pos, dtype=torch.int32, device=DEV)

    def want(self, window=0, sinks=0, scale=None, gated=True):
        s, d = self.s, self.s.D
        out, bound = [], []
        for i, p in enumerate(self.pos):
            pages = self.table[i].tolist()
            there = torch.tensor([0 <= x < self.kpool.shape[0] for x in pages]).repeat_interleave(self.page)
            o, e = po.attend(self.qg[i, :self.new[i], :, :d], po.rows_of(self.kpool, pages, d, self.ki),
                             po.rows_of(self.vpool, pages, d, self.vi), there, p, window, sinks, scale or d ** -0.5,
                             self.qg[i, :self.new[i], :, d:] if gated else None, self.dtype)
            out.append(o), bound.append(e)
        return out, bound

    def check(self, out, window=0, sinks=0, scale=None, gated=True, left=None):
        """out [n_seq, n, heads, d] against the oracle; rows past a sequence's end still hold `left`."""
        out = out.double().cpu()
        for i, (o, e) in enumerate(zip(*self.want(window, sinks, scale, gated))):
            got = out[i, :self.new[i]]
            bad = ~((got - o).abs() <= e)
            assert not bad.any(), (f"sequence {i}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - o).abs().max()):.3e} "
                                   f"at bounds up to {float(e.max()):.3e}, first at {bad.nonzero()[0].tolist()}")
            if left is not None:
                assert (out[i, self.new[i]:] == left).all(), f"rows past sequence {i}'s end were written"


def attend(att, b, window=0, sinks=0, gated=True, **kw):
    d = b.s.D
    kpool, vpool, table, pos = b.dev()
    qg = b.qg.to(DEV)
    out = torch.full((*qg.shape[:3], d), 7.0, dtype=b.dtype, device=DEV)
    att.paged_attend(qg[..., :d], kpool, vpool, table, pos, out, gate=qg[..., d:] if gated else None, lens=b.lens, window=window,
                     sinks=sinks, **kw)
    torch.cuda.synchronize()
    return out


# ---- attention -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,pos,n,page", [
    (TINY, [0], 1, 32), (TINY, [31, 32, 33, 63, 64], 1, 32), (QWEN3_NEXT, [0, 1, 500], 1, 64), (QWEN3_NEXT, [700], 1, 32),
    (D128, [127, 128, 300], 1, 128), (MANY, [95, 260], 1, 64), (EVEN, [200, 3], 1, 64),
    (QWEN3_NEXT, [60, 0, 333], 4, 32), (D128, [10, 64], 5, 64), (EVEN, [29, 61], 8, 32), (TINY, [100], 8, 256),
    (TINY_GGUF, [5, 40], 17, 32), (QWEN3_NEXT, [0, 100], 9, 64), (QWEN3_NEXT, [77], 33, 32), (D128, [0], 131, 32),
    (EVEN, [0, 50], 129, 64), (MANY, [31], 40, 32), (TINY, [3, 0], 200, 64)], ids=str)
def test_attend(contexts, s, pos, n, page, dtype):
    b = Batch(len(pos) * 1000 + n, s, pos, n, page, dtype)
    b.check(attend(contexts(s), b))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,pos,n,page,window,sinks", [
    (QWEN3_NEXT, [500, 3], 1, 64, 64, 4), (QWEN3_NEXT, [500], 1, 32, 1, 0), (D128, [300, 100], 4, 32, 33, 40), (TINY, [1000], 1, 32, 128, 1),
    (TINY, [0, 200], 90, 32, 17, 5), (QWEN3_NEXT, [130], 50, 64, 100, 70), (D128, [400], 70, 32, 64, 0), (EVEN, [64], 150, 64, 1, 1),
    (MANY, [10, 90], 60, 32, 500, 3), (TINY, [700], 3, 64, 1 << 30, 1 << 30)], ids=str)
def test_window_and_sinks(contexts, s, pos, n, page, window, sinks, dtype):
    b = Batch(window + n, s, pos, n, page, dtype)
    b.check(attend(contexts(s), b, window, sinks), window, sinks)


@pytest.mark.parametrize("n", [3, 70])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_ragged_batch_strides_and_rows_left_alone(contexts, n, dtype):
    """Sequences of 0, 1, 2, all and (clamped) more new tokens; garbage in unused rows of q and gate stays unused; out is
    a slice of wider rows whose other columns, like the rows past a sequence's end, keep what they held."""
    s = D128
    b = Batch(n, s, [40, 0, 77, 130, 9, 64], n, 32, dtype, lens=[0, 1, 2, n, n + 50, -3])
    for i, m in enumerate(b.new):
        b.qg[i, m:] = NAN
    kpool, vpool, table, pos = b.dev()
    qg = b.qg.to(DEV)
    wide = torch.full((6, n, s.NH * s.D + 24), 7.0, dtype=dtype, device=DEV)
    out = wide[..., 8:8 + s.NH * s.D].unflatten(-1, (s.NH, s.D))
    wide_table = torch.full((6, table.shape[1] + 3), -5, dtype=torch.int32, device=DEV)
    wide_table[:, :table.shape[1]] = table
    contexts(s).paged_attend(qg[..., :s.D], kpool, vpool, wide_table[:, :table.shape[1]], pos, out, gate=qg[..., s.D:], lens=b.lens)
    b.check(out, left=7)
    assert (wide[..., :8] == 7).all() and (wide[..., 8 + s.NH * s.D:] == 7).all()


@pytest.mark.parametrize("n", [1, 4, 40])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_without_gate_and_with_a_scale(contexts, n, dtype):
    b = Batch(n, QWEN3_NEXT, [100, 31], n, 32, dtype)
    b.check(attend(contexts(QWEN3_NEXT), b, gated=False, scale=0.11), scale=0.11, gated=False)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 60])
def test_hidden_keys_may_hold_anything(contexts, n, dtype):
    """NaN and infinities in the keys and values that no token sees (before the window, in pages given back, behind the last
    row) leave every output as it is; those of a later token of the chunk leave the earlier tokens as they are."""
    s, window, sinks, pos, page = QWEN3_NEXT, 80, 3, 400, 32
    b = Batch(5 + n, s, [pos], n, page, dtype)
    clean = attend(contexts(s), b, window, sinks)
    b.check(clean, window, sinks)
    junk = torch.tensor([NAN, float("inf"), -float("inf"), 65504.0], dtype=F16).repeat(s.D // 4).expand(s.NKV, s.D)
    pages = b.table[0].tolist()
    first = pos - window + 1
    for pool, place in ((b.kpool, b.ki), (b.vpool, b.vi)):
        po.put_rows(pool, pages, s.D, place, range(sinks, first), [junk] * (first - sinks))
    assert torch.equal(attend(contexts(s), b, window, sinks), clean)
    b.table[0, 1:first // page] = torch.tensor([-1, b.kpool.shape[0], 1 << 30, -(1 << 31)] * 8, dtype=torch.int32)[:first // page - 1]
    assert torch.equal(attend(contexts(s), b, window, sinks), clean)
    if n > 2:
        last = pos + n - 1
        for pool, place in ((b.kpool, b.ki), (b.vpool, b.vi)):
            po.put_rows(pool, pages, s.D, place, [last], [junk])
        got = attend(contexts(s), b, window, sinks)
        assert torch.equal(got[:, :n - 1], clean[:, :n - 1])
        assert got[:, n - 1].isnan().any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 4, 60])
def test_keys_without_pages(contexts, n, dtype):
    """Pages that are not there hide their keys; rows that see no key, or lie outside the table's positions, are zero."""
    s, page = D128, 32
    b = Batch(n, s, [200, 200, 150], n, page, dtype)
    b.table[0, 2:5] = torch.tensor([-1, 10 ** 6, -7], dtype=torch.int32)
    b.table[1, :] = -1
    b.table[2, 0] = b.kpool.shape[0]
    out = attend(contexts(s), b)
    b.check(out)
    assert (out[1] == 0).all()
    # a window of 8 whose pages are gone: nothing is left to see
    b.table[0, 6:] = -1
    out = attend(contexts(s), b, 8, 0)
    b.check(out, 8, 0)


@pytest.mark.parametrize("n", [1, 4, 70])
def test_positions_outside_the_table(contexts, n):
    s = TINY
    b = Batch(n, s, [40, 40, 40, 40], n, 32, F32)
    top = b.table.shape[1] * 32
    b.pos = [-3, top - 2, top + 5, 2 ** 31 - 1]
    keys = [po.rows_of(p, b.table[1].tolist(), s.D, i) for p, i in ((b.kpool, b.ki), (b.vpool, b.vi))]
    for pool, rows, place in zip((b.kpool, b.vpool), keys, (b.ki, b.vi)):
        for i in range(4):  # every position of the tables written
            po.put_rows(pool, b.table[i].tolist(), s.D, place, range(top), torch.nan_to_num(rows, nan=0.5))
    out = attend(contexts(s), b)
    b.check(out)
    assert (out[2] == 0).all() and (out[3] == 0).all() and (out[0, :3] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 50])
def test_large_and_small_magnitudes(contexts, n, dtype):
    """Scores over a wide range (a key may take the whole weight, or all share it), keys and values near fp16's largest,
    queries far above fp16's range and far below it."""
    s = QWEN3_NEXT
    for seed, q_sd, k_sd in ((1, 30.0, 8.0), (2, 1e6, 1e-6), (3, 1e-9, 1.0), (4, 1e-3, 2e4)):
        b = Batch(seed, s, [300], n, 64, dtype, keys_sd=k_sd)
        b.kpool = torch.where(b.kpool.isinf(), b.kpool.sign() * 65504, b.kpool)
        b.qg[..., :s.D] = (b.qg[..., :s.D].float() * q_sd).to(dtype)
        b.check(attend(contexts(s), b))


@pytest.mark.parametrize("n,pos", [(1, 900), (4, 900), (100, 700)])
def test_same_bits_on_another_stream_with_own_workspaces_and_in_a_graph(contexts, n, pos):
    """A call's bits do not depend on the stream or on what runs beside it; captured calls replay with new inputs, the
    program's eager calls between the replays."""
    s = QWEN3_NEXT
    att = contexts(s)
    b = Batch(n, s, [pos, pos // 3, 5], n, 64, BF16, lens=[n, max(1, n // 2), n])
    kpool, vpool, table, at = b.dev()
    qg = b.qg.to(DEV)
    want = attend(att, b)
    b.check(want, left=7)
    ws = [torch.full((att.paged_workspace(),), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(2)]
    outs = [torch.full_like(want, 7.0) for _ in range(2)]
    call = lambda i, st=None: att.paged_attend(qg[..., :s.D], kpool, vpool, table, at, outs[i], gate=qg[..., s.D:], lens=b.lens,  # noqa: E731
                                               workspace=ws[i], stream=st)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            call(i, streams[i])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(0)
    first = qg.clone()
    for turn in range(4):
        qg.copy_(first if turn % 2 == 0 else first.flip(1))
        outs[0].fill_(7.0), outs[1].fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        call(1)
        assert torch.equal(outs[0], outs[1])
        if turn % 2 == 0:
            assert torch.equal(outs[0], want)


def test_pages_past_4_gib(contexts):
    """Pages whose bytes lie beyond 32-bit offsets of the pools."""
    s, page = QWEN3_NEXT, 256
    b = Batch(3, s, [700, 300], 5, page, BF16)
    per = s.NKV * page * s.D
    n_pages = (5 << 30) // (2 * per)
    big = [torch.zeros((n_pages, s.NKV, page * s.D), dtype=F16, device=DEV) for _ in "kv"]
    far = torch.arange(n_pages - b.kpool.shape[0], n_pages)
    for x, pool in zip(big, (b.kpool, b.vpool)):
        x[far.to(DEV)] = pool.to(DEV)
    _, _, table, pos = b.dev()
    qg = b.qg.to(DEV)
    out = torch.empty((2, 5, s.NH, s.D), dtype=BF16, device=DEV)
    contexts(s).paged_attend(qg[..., :s.D], *big, (table + int(far[0])).contiguous(), pos, out, gate=qg[..., s.D:])
    b.check(out)
    many = Batch(3, s, [700, 300], 40, page, BF16)
    for x, pool in zip(big, (many.kpool, many.vpool)):
        x[far.to(DEV)] = pool.to(DEV)
    qg = many.qg.to(DEV)
    out = torch.empty((2, 40, s.NH, s.D), dtype=BF16, device=DEV)
    contexts(s).paged_attend(qg[..., :s.D], *big, (many.table.to(DEV) + int(far[0])).contiguous(), many.dev()[3], out,
                             gate=qg[..., s.D:])
    many.check(out)
    del big
    torch.cuda.empty_cache()


# ---- append --------------------------------------------------------------------------------------------------

def rope_table(s, rows):
    freq = s.theta ** -(torch.arange(0, s.R, 2, dtype=torch.float64) / s.R)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).float()


def check_append(att, b, k, v, qn, kn, rope, own_rope=False, with_q=True):
    """Appends b's rows on the GPU; pools bit for bit outside the appended positions, within bounds inside."""
    s, d = b.s, b.s.D
    before = [b.kpool.clone(), b.vpool.clone()]
    kpool, vpool, table, pos = b.dev()
    qg = b.qg.to(DEV)
    q_out = torch.full((*qg.shape[:3], d), 7.0, dtype=b.dtype, device=DEV)
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    att.paged_append(dev(k), dev(v), kpool, vpool, table, pos, q=qg[..., :d] if with_q else None, q_out=q_out if with_q else None,
                     qn=dev(qn), kn=dev(kn), rope=None if own_rope else dev(rope), lens=b.lens)
    got_k, got_v, q_out = kpool.cpu(), vpool.cpu(), q_out.double().cpu()
    limit = min(b.table.shape[1] * b.page, rope.shape[0])
    for i, p in enumerate(b.pos):
        m = b.new[i]
        ok = [t for t in range(m) if 0 <= p + t < limit]
        at = [p + t for t in ok]
        pages = b.table[i].tolist()
        want_k, ek = po.turned(k[i, ok], kn, rope, at, s.eps)
        rows = po.rows_of(got_k, pages, d, b.ki)[at].double() if at else want_k
        put = torch.tensor([0 <= pages[x // b.page] < b.kpool.shape[0] for x in at], dtype=torch.bool)
        err = (rows - want_k).abs()[put]
        assert (err <= (1.01 * ek + po.HALF[F16] * (want_k.abs() + ek) + 2.0 ** -25)[put]).all(), float(err.max())
        rows = po.rows_of(got_v, pages, d, b.vi)[at] if at else rows
        assert torch.equal(rows[put], v[i, ok].to(F16)[put])
        for pool, got, place in ((before[0], got_k, b.ki), (before[1], got_v, b.vi)):
            if at:
                now = po.rows_of(got, pages, d, place)[at]
                po.put_rows(pool, pages, d, place, at, now)
        if with_q:
            want_q, eq = po.turned(b.qg[i, ok, :, :d], qn, rope, at, s.eps)
            err = (q_out[i, ok] - want_q).abs()
            assert (err <= 1.01 * eq + po.HALF[b.dtype] * (want_q.abs() + eq) + 1e-37).all(), float(err.max())
            gone = [t for t in range(m) if t not in ok]
            assert (q_out[i, gone] == 0).all() and (q_out[i, m:] == 7).all()
    for pool, got in zip(before, (got_k, got_v)):
        assert torch.equal(pool.view(torch.int16), got.view(torch.int16)), "memory outside the appended rows changed"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s,pos,n,page,lens", [
    (TINY, [0], 1, 32, None), (QWEN3_NEXT, [31, 100, 0], 1, 32, None), (D128, [5, 64], 4, 64, [4, 0]), (MANY, [33], 9, 32, None),
    (EVEN, [7, 8, 1], 17, 32, [17, 30, 3]), (QWEN3_NEXT, [60, 3], 100, 64, [100, 41]), (TINY_GGUF, [250], 20, 256, None)], ids=str)
def test_append(contexts, s, pos, n, page, lens, dtype):
    b = Batch(n + 7, s, pos, n, page, dtype, lens)
    k, v = (b.r(len(pos), n, s.NKV, s.D).to(dtype) for _ in "kv")
    for i, m in enumerate(b.new):
        k[i, m:], v[i, m:], b.qg[i, m:] = NAN, NAN, NAN
    check_append(contexts(s), b, k, v, b.r(s.D, sd=0.1), b.r(s.D, sd=0.1), rope_table(s, 1024))


def test_append_variants(contexts):
    """Without norms, without queries, with the context's rope table, strided k and v, positions past the tables."""
    s = D128
    att = contexts(s)
    for kw in ({}, {"own_rope": True}, {"with_q": False}):
        b = Batch(3, s, [30, -5, 300], 40, 32, F32, lens=[40, 40, 37])
        b.table = b.table[:, :10]  # 320 positions: the last sequence's rows pass them
        b.table[0, 1] = -1
        rope = att.rope_table().cpu()[:310].contiguous() if not kw.get("own_rope") else att.rope_table().cpu()
        rows = b.r(3, 40, 2 * s.NKV, s.D)
        check_append(att, b, rows[:, :, :s.NKV], rows[:, :, s.NKV:], None, None, rope, **kw)
        check_append(att, b, rows[:, :, :s.NKV], rows[:, :, s.NKV:], b.r(s.D, sd=0.1), None, rope, **kw)


# ---- together ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("s,dtype", [(QWEN3_NEXT, F32), (D128, BF16), (TINY, F32)], ids=["next", "d128", "tiny"])
def test_serving_loop(contexts, s, dtype):
    """Two requests of different ages through prompt chunks, a verify pass whose last drafts are rejected, decode steps and an
    idle place, each pass an append and an attend: every output against the 64-bit attention over all rows so far."""
    att = contexts(s)
    g = torch.Generator().manual_seed(1)
    r = lambda *shape, sd=1.0: torch.randn(shape, generator=g) * sd  # noqa: E731
    page, pages, b = 32, 8, 3
    d = s.D
    table = torch.randperm(b * pages, generator=g).view(b, pages).to(torch.int32).to(DEV)
    kpool = torch.full((b * pages, s.NKV, page * d), NAN, dtype=F16, device=DEV)
    vpool = kpool.clone()
    qn, kn = r(d, sd=0.1), r(d, sd=0.1)
    ki, vi = po.block_places(d)
    pos, ws = [0, 0, 0], torch.empty(att.paged_workspace(), dtype=torch.uint8, device=DEV)
    for n, lens, keep in ((70, [70, 33, 0], [70, 33, 0]), (20, [20, 7, 0], [20, 7, 0]), (4, [4, 4, 0], [2, 4, 0]), (1, [1, 1, 0], [1, 1, 0]),
                          (1, [1, 0, 1], [1, 0, 1])):
        qg, k, v = r(b, n, s.NH, 2 * d).to(dtype), r(b, n, s.NKV, d).to(dtype), r(b, n, s.NKV, d).to(dtype)
        q_out = torch.zeros(b, n, s.NH, d, dtype=dtype, device=DEV)
        out = torch.full_like(q_out, 7.0)
        at, ln = torch.tensor(pos, dtype=torch.int32, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
        rows = qg.to(DEV)
        att.paged_append(k.to(DEV), v.to(DEV), kpool, vpool, table, at, q=rows[..., :d], q_out=q_out, qn=qn.to(DEV), kn=kn.to(DEV), lens=ln)
        att.paged_attend(q_out, kpool, vpool, table, at, out, gate=rows[..., d:], lens=ln, workspace=ws)
        torch.cuda.synchronize()
        kc, vc, qc = kpool.cpu(), vpool.cpu(), q_out.cpu()
        for i in range(b):
            m = lens[i]
            own = table[i].tolist()
            o, e = po.attend(qc[i, :m], po.rows_of(kc, own, d, ki), po.rows_of(vc, own, d, vi), torch.ones(pages * page, dtype=torch.bool),
                             pos[i], 0, 0, d ** -0.5, qg[i, :m, :, d:], dtype)
            assert ((out[i, :m].double().cpu() - o).abs() <= e).all()
            assert (out[i, m:] == 7).all()
            pos[i] += keep[i]
