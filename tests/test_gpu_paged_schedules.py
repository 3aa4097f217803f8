"""Paged attention at sizes where its schedules cut sequences: several blocks a wave, parts of unequal length, equal runs that end
in one sequence and begin in the next, batches of more sequences than a wave has lanes, more items than the plan has threads.
Each case asserts, from a restatement of the schedule, that it takes the way it is meant for.

Two checks see a block of keys that is lost or taken twice, which the worst-case bounds of thousands of keys hide:
  - queries of zero: every weight is the same power of two, every block has dims of its own, and the outputs are known
    but for the quotient's roundings;
  - ordinary queries: the 2-norm of a token's error against 64 bits, 2^-8 of the output in bf16 (its roundings alone at most) and
    2^-18 in fp32 (64 roundings' worth); 32 of 35,000 keys are 2^-5 of it."""
import pytest
import torch

import paged_oracle as po
from common import TINY, QWEN3_NEXT, D128
from test_gpu_paged import BF16, DEV, EVEN, F16, F32, MANY, contexts  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


# ---- the schedules, restated -----------------------------------------------------------------------------------

def ceil_div(a, b):
    return -(-a // b)


def tiles(pos, t0, t1, size, limit, window, sinks):
    """Tiles of `size` keys that some of tokens [t0, t1) sees."""
    if t0 >= t1:
        return 0
    lo, hi = max(pos + t0, 0), min(pos + t1, limit) - 1
    if lo > hi:
        return 1
    first = max(lo - window + 1, 0) // size if window else 0
    return min(ceil_div(sinks, size), first) + hi // size + 1 - first


def few_schedule(units, nkv, groups):
    """("parts", units of the longest part, parts unequal within a sequence) or ("runs", units a run, sequences cut by a run's end)"""
    total = sum(units) * nkv
    run = max(1, ceil_div(total, groups))
    if len(units) <= 64:
        for spare in range(4):
            parts = [ceil_div(u, run + spare) for u in units]
            if sum(parts) * nkv <= groups:
                return "parts", max(ceil_div(u, p) for u, p in zip(units, parts) if u), sum(u % p > 0 for u, p in zip(units, parts) if u)
    at, cut = 0, 0
    for _ in range(nkv):
        for u in units:
            cut += u > 0 and at // run != (at + u - 1) // run
            at += u
    return "runs", run, cut


def plan_cuts(counts, nkv, groups):
    """Items that the plan's equal runs cut inside (runs of more items than threads, where equal parts are not tried)"""
    cost = sum(c + 4 for c in counts if c)
    run, at, cut = max(1, ceil_div(cost * nkv, groups)), 0, 0
    near = run // 12
    for _ in range(nkv):
        for c in counts:
            if c:
                offs = [w * run - at - 4 for w in range(ceil_div(at, run), ceil_div(at + 4 + c, run))]
                cut += any(near < x < c - near for x in offs)
                at += c + 4
    return cut


# ---- batches whose sequences share the pages of a small pool, each in an order of its own ------------------------

class Shared:
    def __init__(self, seed, s, pos, new, n, page, dtype, window=0, sinks=0):
        self.s, self.pos, self.new, self.n, self.page, self.dtype, self.window, self.sinks = s, pos, new, n, page, dtype, window, sinks
        g = torch.Generator().manual_seed(seed)
        self.count = count = max(ceil_div(p + n, page) for p in pos)  # pages of a sequence, and of the pool
        self.g, self.limit = g, count * page
        self.table = (torch.arange(count)[None] + 5 * torch.arange(len(pos))[:, None]) % count  # page (i + 5 b) of the pool
        self.krows = torch.randn(count * page, s.NKV, s.D, generator=g).to(F16)
        self.vrows = torch.randn(count * page, s.NKV, s.D, generator=g).to(F16)
        self.q = torch.randn(len(pos), n, s.NH, s.D, generator=g).to(dtype)
        self.gate = torch.randn(len(pos), n, s.NH, s.D, generator=g).to(dtype)

    def units(self):
        return [ceil_div(tiles(p, 0, m, 32, self.limit, self.window, self.sinks), 4) for p, m in zip(self.pos, self.new)]

    def counts(self, tok):
        return [tiles(p, t, min(t + tok, m), 64, self.limit, self.window, self.sinks) for p, m in zip(self.pos, self.new) for t in range(0, self.n, tok)]

    def pool(self, rows, place):
        s = self.s
        pool = torch.empty(self.count, s.NKV, self.page // 32, 32 * s.D, dtype=F16)
        pool[..., place.flatten()] = rows.view(self.count, self.page // 32, 32, s.NKV, s.D).permute(0, 3, 1, 2, 4).flatten(-2)
        return pool.flatten(2).to(DEV)

    def own(self, rows, b):
        """The rows of sequence b by its positions."""
        return rows.view(self.count, self.page, self.s.NKV, -1)[self.table[b]].flatten(0, 1)

    def run(self, att, q, gate):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        ki, vi = po.block_places(self.s.D)
        out = torch.full(q.shape, 7.0, dtype=self.dtype, device=DEV)
        att.paged_attend(q.to(DEV), self.pool(self.krows, ki), self.pool(self.vrows, vi), self.table.to(torch.int32).to(DEV), i32(self.pos), out,
                         gate=None if gate is None else gate.to(DEV), lens=i32(self.new), window=self.window, sinks=self.sinks)
        out = out.double().cpu()
        for b, m in enumerate(self.new):
            assert (out[b, m:] == 7).all(), f"rows past sequence {b}'s end were written"
        return out

    def check_blocks(self, att):
        """Queries of zero: the mean of the values that a token sees, block i of the pool 1 to 3 in dim i (mod D), 0 elsewhere."""
        s = self.s
        block = torch.arange(self.count * self.page) // 32
        self.vrows = torch.zeros(self.count * self.page, s.NKV, s.D, dtype=F16)
        for h in range(s.NKV):
            self.vrows[torch.arange(len(block)), h, (block + 7 * h) % s.D] = (1 + (block // s.D + h) % 3).to(F16)
        out = self.run(att, torch.zeros_like(self.q), None).unflatten(2, (s.NKV, s.G))
        for b, (p, m) in enumerate(zip(self.pos, self.new)):
            sums = torch.cat([torch.zeros(1, s.NKV, s.D, dtype=torch.float64), self.own(self.vrows, b).double().cumsum(0)])
            at = p + torch.arange(m)
            first = (at - self.window + 1).clamp(min=0) if self.window else torch.zeros_like(at)
            kept = first.clamp(max=self.sinks)
            seen = at + 1 - first + kept
            want = (sums[at + 1] - sums[first] + sums[kept]) / seen[:, None, None]
            # sums of weights (2^8) and of weighted values stay below 2^24 and are exact; the reciprocal and the product
            assert m == 0 or int(max(seen.max(), (want * seen[:, None, None]).max())) < 1 << 16
            bound = (3 * po.EPS32 + po.HALF[self.dtype] * (1 + 3 * po.EPS32)) * want
            err = (out[b, :m] - want[:, :, None]).abs()
            bad = err > bound[:, :, None]
            assert not bad.any(), f"sequence {b}: {int(bad.sum())} outputs off, first at {bad.nonzero()[0].tolist()}"

    def check_norms(self, att, sequences, tokens):
        """Ordinary queries: each token's outputs against 64 bits as a 2-norm, at some sequences and tokens."""
        s = self.s
        out = self.run(att, self.q, self.gate)
        for b in sequences:
            k, v = self.own(self.krows, b), self.own(self.vrows, b)
            for t in sorted({x for x in tokens if x < self.new[b]}):
                want, _ = po.attend(self.q[b, t:t + 1], k, v, torch.ones(len(k), dtype=torch.bool), self.pos[b] + t, self.window, self.sinks,
                                    s.D ** -0.5, self.gate[b, t:t + 1], self.dtype)
                far = float((out[b, t] - want[0]).norm() / want[0].norm())
                assert far <= (2.0 ** -8 if self.dtype is BF16 else 2.0 ** -18), f"sequence {b}, token {t}: {far:.2e}"


def ragged(count, top, seed):
    g = torch.Generator().manual_seed(seed)
    return (top * (0.1 + 0.9 * torch.rand(count, generator=g))).int().tolist()


# (heads, positions so far, most new tokens, page, window, sinks), the way the schedule takes and its least units a workgroup
FEW = [
    ("parts of several units", (MANY, [10000, 9000, 10500, 7001], 1, 64, 0, 0), "parts", 4),
    ("the same, four tokens", (EVEN, [10000, 6100], 4, 32, 0, 0), "parts", 2),
    ("parts behind a window", (MANY, [30000, 25001, 28000, 27777], 2, 64, 12000, 300), "parts", 4),
    ("parts of one KV head", (QWEN3_NEXT, [33000, 20011, 30000], 4, 128, 0, 0), "parts", 3),
    ("runs, uneven ages", (QWEN3_NEXT, ragged(50, 16000, 1), 1, 128, 0, 0), "runs", 16),
    ("runs of a few tokens", (MANY, ragged(60, 9000, 2), 8, 64, 0, 0), "runs", 20),
    ("runs of two tiles of 256 dims", (QWEN3_NEXT, ragged(70, 4000, 8), 4, 32, 0, 0), "runs", 8),
    ("runs behind a window", (MANY, ragged(50, 9000, 3), 2, 32, 7000, 70), "runs", 16),
    ("more sequences than lanes", (MANY, ragged(70, 3000, 4), 1, 64, 0, 0), "runs", 10),
    ("two and three a lane", (TINY, ragged(130, 3000, 5), 3, 32, 0, 0), "runs", 3),
    ("more behind a window", (D128, ragged(100, 3000, 6), 2, 32, 1000, 5), "runs", 2),
    ("parts of over 64 blocks a wave", (EVEN, [40000] * 16, 1, 128, 0, 0), "parts", 65),
    ("runs of over 64 blocks a wave", (EVEN, ragged(130, 16000, 7), 1, 128, 0, 0), "runs", 100),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case,way,least", [c[1:] for c in FEW], ids=[c[0] for c in FEW])
def test_few_tokens(contexts, case, way, least, dtype):  # noqa: F811
    s, pos, n, page, window, sinks = case
    lens = [n - (i % 3 == 1) * (i % n) for i in range(len(pos))]
    if len(pos) > 20:
        lens[3] = lens[17] = 0
    b = Shared(len(pos), s, pos, lens, n, page, dtype, window, sinks)
    assert n * s.G <= 32
    groups = torch.cuda.get_device_properties(0).multi_processor_count * (1 if s.D == 256 else 2)
    taken, units, cut = few_schedule(b.units(), s.NKV, groups)
    assert (taken, cut > 0) == (way, True) and units >= least, (taken, units, cut)
    att = contexts(s)
    b.check_norms(att, range(0, len(pos), 1 + len(pos) // 4), {0, n - 1})
    b.check_blocks(att)


# ... of chunks, and whether items are joined by a second launch, by the wave that arrives last, or planned by threads of several items
CHUNKS = [
    ("few items, many parts", (EVEN, [20000], 512, 128, 0, 0), "joined"),
    ("one item of a head", (QWEN3_NEXT, [15000], 30, 64, 0, 0), "joined"),
    ("equal parts or runs", (MANY, [9000, 300, 4000], 500, 64, 0, 0), "plan"),
    ("equal runs", (QWEN3_NEXT, [3000], 2048, 64, 0, 0), "plan"),
    ("equal runs behind a window", (D128, [9000, 4000], 3500, 64, 5000, 200), "plan"),
    ("more items than threads", (TINY, [15000 if i % 211 == 7 else 7 * i % 90 for i in range(1100)], 33, 64, 0, 0), "threads"),
    ("more items behind a window", (TINY, [16000 if i % 300 == 7 else 7 * i % 90 for i in range(1300)], 40, 64, 9000, 130), "threads"),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case,way", [c[1:] for c in CHUNKS], ids=[c[0] for c in CHUNKS])
def test_chunks(contexts, case, way, dtype):  # noqa: F811
    s, pos, n, page, window, sinks = case
    lens = [n - (i % 3 == 1) * (i % n) for i in range(len(pos))]
    if len(pos) > 20:
        lens[3] = lens[400] = 0
    b = Shared(n, s, pos, lens, n, page, dtype, window, sinks)
    groups = torch.cuda.get_device_properties(0).multi_processor_count & ~7
    tok = (128 if s.D == 256 and dtype is F32 else 256) // s.G
    pairs = len(pos) * ceil_div(n, tok)
    assert way == ("joined" if pairs * s.NKV * 4 <= groups and pairs <= 64 else "threads" if pairs > 1024 else "plan")
    if way == "threads":
        assert plan_cuts(b.counts(tok), s.NKV, groups) > 3
    att = contexts(s)
    long = [i for i, p in enumerate(pos) if p > 2000]
    b.check_norms(att, long[:3] + [0, len(pos) - 1], {0, 1, n // 2, n - 1})
    b.check_blocks(att)
