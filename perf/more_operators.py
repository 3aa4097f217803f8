"""The full-attention layers' operators for batches of sequences over a paged K/V cache, as timed cases.

A case is one pass of one operator over one layer. Kinds:
  append  new tokens of n_seq sequences: QK norm and position rotation, keys and values into their pages, queries out
  attend  attention of those tokens over their sequences' pages: one token a sequence (decode), a few (speculative
          verify) or a chunk of a prompt, causal, with a sigmoid gate; with a window each token sees its last
          `window` positions and the first `sinks`

The caches are pools of pages [n_pages, KV heads, page * head dim] fp16 in blocks of 32 positions (include/qwattn.h),
table [n_seq, pages] says which page holds positions page * i and on, pos [n_seq] how many tokens a sequence has
already. With `own` false, run() computes the operators from elementary torch operations in fp32; with `own` true it
calls the package. exact() restates them in fp64, sequence by sequence and head by head.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
EPS, THETA, MAX_CTX = 1e-6, 1e7, 40960
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# (query heads, KV heads, head dim, rotated dims)
NEXT, D128, TINY, MANY, EVEN = (16, 2, 256, 64), (8, 2, 128, 32), (4, 1, 64, 16), (32, 8, 128, 128), (8, 8, 64, 64)


# ---- cases -------------------------------------------------------------------------------------------------

def case(kind, n_seq, n, pos, dtype, heads=NEXT, page=64, ragged=False, window=0, sinks=0):
    """n_seq sequences with up to n new tokens each behind up to pos cached ones (ragged: fewer, sequence by sequence)."""
    nh, nkv, d, r = heads
    c = {"kind": kind, "n_seq": n_seq, "n": n, "pos": pos, "dtype": dtype, "heads": nh, "kv_heads": nkv, "dim": d,
         "rope": r, "page": page, "ragged": ragged}
    return c | ({"window": window, "sinks": sinks} if kind == "attend" else {})


def listed():
    return [
        # a decode step of one sequence: launch and latency
        {"name": "append_decode", **case("append", 1, 1, 1000, "f32")},
        # a batch of prompt chunks of different lengths
        {"name": "append_chunks_4x1k", **case("append", 4, 1024, 2000, "bf16", ragged=True)},
        # a decode step early in a conversation: the smallest attention call
        {"name": "decode_500", **case("attend", 1, 1, 500, "f32")},
        # a decode step of one long sequence, split over the chip
        {"name": "decode_32k", **case("attend", 1, 1, 32767, "f32")},
        # a decode step of a serving batch, requests of different ages
        {"name": "decode_batch_32", **case("attend", 32, 1, 16000, "bf16", page=128, ragged=True)},
        # speculative verify of a batch: one token and three drafts
        {"name": "verify_8x4", **case("attend", 8, 4, 8190, "f32", page=32, ragged=True)},
        # decode with a sliding window and a few first tokens kept, past many pages that no token sees any more
        {"name": "window_decode_16", **case("attend", 16, 1, 32000, "bf16", ragged=True, window=4096, sinks=4)},
        # a few tokens more than a verify, on a long context: few rows, a long key axis
        {"name": "chunk_61_on_16k", **case("attend", 1, 61, 16384, "f32", page=32)},
        # a batch of short prompts of odd lengths from their first token on, another head layout
        {"name": "prompts_6x700", **case("attend", 6, 701, 0, "f32", D128, page=32, ragged=True)},
        # a chunk of a long prompt, bf16 activations
        {"name": "chunk_2k_on_2k", **case("attend", 1, 2048, 2048, "bf16")},
        # the same work from fp32 activations, as the projections give them
        {"name": "chunk_1k_on_7k", **case("attend", 1, 1024, 7168, "f32", page=256)},
        # a long chunk through a layer with a sliding window
        {"name": "window_chunk_4k", **case("attend", 1, 4096, 8192, "bf16", window=1024, sinks=64)},
    ]


def spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    form = lambda c: c["kind"] + ("_few" if c["kind"] == "attend" and c["n"] <= 8 else "")  # noqa: E731
    top = {}
    for c in listed():
        w, (b, f) = work(c), top.get(form(c), (0, 0))
        top[form(c)] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        kind = rng.choice(["append", "attend", "attend", "attend"])
        few = rng.random() < 0.5
        heads, dtype = rng.choice([NEXT, NEXT, D128, TINY, MANY, EVEN]), rng.choice(["f32", "bf16"])
        page, ragged = rng.choice([32, 64, 64, 128, 256]), rng.random() < 0.5
        if few:
            c = case(kind, rng.choice([1, spread(rng, 1, 48)]), spread(rng, 1, 8), spread(rng, 1, 32000), dtype, heads, page, ragged)
        else:
            c = case(kind, rng.choice([1, spread(rng, 1, 8)]), spread(rng, 9, 4096), rng.choice([0, spread(rng, 1, 32000)]), dtype,
                     heads, page, ragged)
        if kind == "attend" and rng.random() < 0.4:
            c |= {"window": spread(rng, 1, 8192), "sinks": rng.choice([0, 1, 4, spread(rng, 1, 200)])}
        w, most = work(c), top[form(c)]
        pool = 4 * c["n_seq"] * (c["pos"] + c["n"]) * c["kv_heads"] * c["dim"]
        # no drawn case costs more than the largest listed one of its form, nor has caches over 2 GiB
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and pool <= 1 << 31 and c not in ({k: v for k, v in x.items() if k != "name"} for x in listed()):
            return c


def lengths(c, seed=None):
    """(tokens already cached, new tokens) of every sequence; seed None: their expectation, for work()."""
    b, n, pos = c["n_seq"], c["n"], c["pos"]
    if not c["ragged"]:
        return [pos] * b, [n] * b
    if seed is None:
        return [int(pos * (0.1 + 0.9 * (i + 0.5) / b)) for i in range(b)], [max(1, int(n * (0.1 + 0.9 * (i + 0.5) / b))) for i in range(b)]
    g = torch.Generator().manual_seed(seed)
    share = 0.1 + 0.9 * torch.rand(2, b, generator=g, dtype=torch.float64)
    return [int(pos * s) for s in share[0].tolist()], [max(1, int(n * s)) for s in share[1].tolist()]


def work(c):
    size = 2 if c["dtype"] == "bf16" else 4
    pos, new = lengths(c)
    rows = sum(new)
    nh, nkv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "append":
        return {"bytes": rows * (size * d * (2 * nh + 2 * nkv) + 4 * nkv * d + 4 * c["rope"]) + 8 * d,
                "flops": rows * d * (nh + nkv) * 8}
    keys, pairs = 0, 0
    for p, m in zip(pos, new):
        if c["window"]:
            first = max(0, p - c["window"] + 1)  # of the first new token's window
            keys += p + m - first + min(c["sinks"], first)
            for q in range(p, p + m):
                start = max(0, q - c["window"] + 1)
                pairs += q + 1 - start + min(c["sinks"], start)
        else:
            keys += p + m
            pairs += m * p + m * (m + 1) // 2
    return {"bytes": 4 * keys * nkv * d + 3 * rows * nh * d * size, "flops": 4 * pairs * nh * d}


# ---- inputs ------------------------------------------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape, sd=1.0):
        return torch.randn(shape, generator=g, device=DEV) * sd

    b, n, nh, nkv, d, page = c["n_seq"], c["n"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    pos, new = lengths(c, seed)
    s = {"case": c}
    # every sequence's pages in any order over the pool, a few pages of nobody between them
    pages = -(-(c["pos"] + n) // page)
    n_pages = b * pages + 3
    s["table"] = torch.randperm(n_pages, generator=g, device=DEV)[:b * pages].view(b, pages).to(torch.int32)
    s["pos"] = torch.tensor(pos, dtype=torch.int32, device=DEV)
    s["lens"] = torch.tensor(new, dtype=torch.int32, device=DEV) if c["ragged"] else None
    s["kpool"], s["vpool"] = (torch.randn((n_pages, nkv, page * d), generator=g, device=DEV, dtype=torch.float16) for _ in "kv")
    # a projection's rows: each query head's query, then its gate
    s["qg"] = normal(b, n, nh, 2 * d).to(dt)
    if c["kind"] == "append":
        s["k"], s["v"] = normal(b, n, nkv, d).to(dt), normal(b, n, nkv, d).to(dt)
        s["qn"], s["kn"] = normal(d, sd=0.1), normal(d, sd=0.1)
        freq = (THETA ** -(torch.arange(0, c["rope"], 2, device=DEV, dtype=torch.float64) / c["rope"]))
        angle = torch.arange(pages * page, device=DEV, dtype=torch.float64)[:, None] * freq
        s["rope"] = torch.stack([torch.cos(angle), torch.sin(angle)], -1).float()
        s["q_out"] = torch.zeros((b, n, nh, d), device=DEV, dtype=dt)
    else:
        s["q"] = normal(b, n, nh, d, sd=1.2).to(dt)
        s["out"] = torch.zeros((b, n, nh, d), device=DEV, dtype=dt)
    return s


# ---- a pass ------------------------------------------------------------------------------------------------

def package():
    """qwen3-local-test_amd as the module qwattn_amd (its folder's name has a hyphen: loaded by path)."""
    if "qwattn_amd" not in sys.modules:
        pkg = os.path.join(ROOT, "qwen3-local-test_amd")
        spec = importlib.util.spec_from_file_location("qwattn_amd", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        sys.modules["qwattn_amd"] = mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    return sys.modules["qwattn_amd"]


_contexts = {}


def context(c):
    """The program's context of a head layout, made at its first call, and the workspace it keeps beside it."""
    heads = c["heads"], c["kv_heads"], c["dim"], c["rope"]
    if heads not in _contexts:
        att = package().Attention(*heads, rope_theta=THETA, max_ctx=MAX_CTX, max_tokens=64, rms_eps=EPS)
        _contexts[heads] = att, torch.empty(att.paged_workspace(), dtype=torch.uint8, device=DEV)
    return _contexts[heads]


def run(s):
    c = s["case"]
    d = c["dim"]
    if own:
        att, workspace = context(c)
        if c["kind"] == "append":
            att.paged_append(s["k"], s["v"], s["kpool"], s["vpool"], s["table"], s["pos"], q=s["qg"][..., :d],
                             q_out=s["q_out"], qn=s["qn"], kn=s["kn"], rope=s["rope"], lens=s["lens"])
            return {"kpool": s["kpool"], "vpool": s["vpool"], "q": s["q_out"]}
        att.paged_attend(s["q"], s["kpool"], s["vpool"], s["table"], s["pos"], s["out"], gate=s["qg"][..., d:],
                         lens=s["lens"], window=c["window"], sinks=c["sinks"], workspace=workspace)
        return {"out": s["out"]}
    return (plain_append if c["kind"] == "append" else plain_attend)(s)


def places(d):
    """Where a block keeps key or value (position kb, dim) of its 32 x d: two [32, d] index tables."""
    kb, e = torch.arange(32, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    k = (((e // 32 * 2 + kb // 4 % 2) * 4 + e // 8 % 4) * 16 + kb // 8 * 4 + kb % 4) * 8 + e % 8
    v = ((e // 16 * 4 + kb // 8) * 16 + e % 16) * 8 + kb % 8
    return k, v


def plain_append(s):
    c = s["case"]
    d, r, page, nkv, (b, n) = c["dim"], c["rope"], c["page"], c["kv_heads"], s["k"].shape[:2]
    p = s["pos"].long()[:, None] + torch.arange(n, device=DEV)
    cs = s["rope"][p][:, :, None]

    def turned(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w)
        lo, hi, cos, sin = y[..., :r // 2], y[..., r // 2:r], cs[..., 0], cs[..., 1]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, y[..., r:]], -1)

    there = torch.arange(n, device=DEV) < (s["lens"][:, None] if s["lens"] is not None else n)
    there = there.expand(b, n)
    seq, tok = torch.nonzero(there, as_tuple=True)
    at = p[seq, tok]
    start = s["table"][seq, at // page].long() * (nkv * page * d) + at % page // 32 * (32 * d)
    start = start[:, None, None] + torch.arange(nkv, device=DEV)[:, None] * (page * d)
    for pool, rows, place in zip((s["kpool"], s["vpool"]), (turned(s["k"], s["kn"]), s["v"].float()), places(d)):
        pool.view(-1)[start + place[at % 32][:, None]] = rows[seq, tok].to(torch.float16)
    q = turned(s["qg"][..., :d], s["qn"]).to(s["q_out"].dtype)
    s["q_out"].copy_(torch.where(there[..., None, None], q, s["q_out"]))
    return {"kpool": s["kpool"], "vpool": s["vpool"], "q": s["q_out"]}


def plain_attend(s):
    c = s["case"]
    d, page, nh, nkv, (b, n) = c["dim"], c["page"], c["heads"], c["kv_heads"], s["q"].shape[:2]
    ki, vi = places(d)
    pages = s["table"].long()
    if c["window"]:  # pages behind every token's window are not read
        first = torch.clamp(s["pos"].long() - c["window"] + 1, min=0) // page
        kept, span = -(-c["sinks"] // page), -(-(c["window"] + n) // page) + 1
        at = torch.cat([torch.arange(kept, device=DEV).expand(b, kept), torch.clamp(first, min=kept)[:, None] + torch.arange(span, device=DEV)], 1)
        key = (at[:, :, None] * page + torch.arange(page, device=DEV)).flatten(1)
        pages = torch.gather(pages, 1, torch.clamp(at, max=pages.shape[1] - 1))
    else:
        key = torch.arange(pages.shape[1] * page, device=DEV).expand(b, -1)

    def rows(pool, place):  # [b, nkv, keys, d]
        x = pool[pages].view(b, -1, nkv, page // 32, 32 * d)[..., place]
        return x.transpose(1, 2).reshape(b, nkv, -1, d).float()

    p = s["pos"].long()[:, None] + torch.arange(n, device=DEV)
    end = (s["pos"] + (s["lens"] if s["lens"] is not None else n)).long()
    sees = key[:, None] <= p[..., None]
    if c["window"]:
        sees &= (key[:, None] > p[..., None] - c["window"]) | (key[:, None] < c["sinks"])
    sees &= key[:, None] < end[:, None, None]
    k, v = rows(s["kpool"], ki), rows(s["vpool"], vi)
    q = s["q"].float().unflatten(2, (nkv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [b, nkv, group * n, d]
    score = (q @ k.transpose(2, 3).contiguous() * d ** -0.5).unflatten(2, (-1, n))
    score = torch.where(sees[:, None, None], score, -math.inf)
    top = torch.clamp(score.amax(-1, keepdim=True), min=torch.finfo(torch.float32).min)
    w = torch.exp(score - top)
    o = (w.flatten(2, 3) @ v) / w.flatten(2, 3).sum(-1, keepdim=True)
    o = o.unflatten(2, (-1, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    o = (o * torch.sigmoid(s["qg"][..., d:].float())).to(s["out"].dtype)
    if s["lens"] is None:
        return {"out": o}
    there = torch.arange(n, device=DEV) < s["lens"][:, None]
    return {"out": torch.where(there[..., None, None], o, s["out"])}


# ---- the definition in fp64 ----------------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    b, n, nh, nkv, d, page, r = c["n_seq"], c["n"], c["heads"], c["kv_heads"], c["dim"], c["page"], c["rope"]
    pos, new = lengths(c, seed)
    e, kb = torch.meshgrid(torch.arange(d, device=DEV), torch.arange(32, device=DEV), indexing="ij")
    inside = {"k": torch.empty(32 * d, dtype=torch.long, device=DEV), "v": torch.empty(32 * d, dtype=torch.long, device=DEV)}
    # the block's element -> position * d + dim
    inside["k"][((e // 32) * 1024 + ((kb // 4) % 2) * 512 + ((e // 8) % 4) * 128 + (kb // 8) * 32 + (kb % 4) * 8 + e % 8).flatten()] = (kb * d + e).flatten()
    inside["v"][((e // 16) * 512 + (kb // 8) * 128 + (e % 16) * 8 + kb % 8).flatten()] = (kb * d + e).flatten()

    if c["kind"] == "append":
        kpool, vpool = (s[m].double().view(-1, nkv, page // 32, 32 * d) for m in ("kpool", "vpool"))
        q_out = s["q_out"].double()

        def turned(x, w, p):
            x = x.double()
            y = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * (1 + w.double())
            cos, sin = s["rope"][p].double().unbind(-1)
            z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * torch.complex(cos, sin)[:, None]
            return torch.cat([z.real, z.imag, y[..., r:]], -1)

        to = {m: torch.argsort(inside[m]).view(32, d) for m in "kv"}
        for i in range(b):
            p = pos[i] + torch.arange(new[i], device=DEV)
            q_out[i, :new[i]] = turned(s["qg"][i, :new[i], :, :d], s["qn"], p)
            where = s["table"][i].long()[p // page]
            for pool, rows, m in ((kpool, turned(s["k"][i, :new[i]], s["kn"], p), "k"), (vpool, s["v"][i, :new[i]].double(), "v")):
                for h in range(nkv):
                    pool[where[:, None], h, (p % page // 32)[:, None], to[m][p % 32]] = rows[:, h]
        return {"kpool": kpool.view(s["kpool"].shape), "vpool": vpool.view(s["vpool"].shape), "q": q_out}

    out = s["out"].double()
    for i in range(b):
        total = pos[i] + new[i]
        mine = s["table"][i, :-(-total // page)].long()
        j, t = torch.arange(total, device=DEV), pos[i] + torch.arange(new[i], device=DEV)[:, None]
        hidden = j > t
        if c["window"]:
            hidden |= (j <= t - c["window"]) & (j >= c["sinks"])
        for h in range(nkv):
            k, v = (torch.empty((mine.numel() * (page // 32), 32 * d), dtype=torch.float64, device=DEV).index_copy_(
                1, inside[m], s[m + "pool"][mine, h].double().view(-1, 32 * d)).view(-1, d)[:total] for m in "kv")
            kt = k.t().contiguous()
            for head in range(h * (nh // nkv), (h + 1) * (nh // nkv)):
                score = (s["q"][i, :new[i], head].double() @ kt / math.sqrt(d)).masked_fill_(hidden, -math.inf)
                out[i, :new[i], head] = torch.softmax(score, -1) @ v / (1 + torch.exp(-s["qg"][i, :new[i], head, d:].double()))
    return {"out": out}
