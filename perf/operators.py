"""The linear-attention and mixture-of-experts operators beside the full-attention layers, as timed cases.

A case is one pass of one operator over the inputs of one layer. Kinds:
  conv    short causal depthwise convolution + SiLU over the rows of n_seq sequences, its last rows carried
  delta   gated delta rule: n tokens of n_seq sequences through a recurrent state [key dim, value dim] a head
  route   the router: the top_k experts of each token's logits, with their softmax weights
  moe     SwiGLU experts in planar Q8_0 over the tokens that a router sent them

With `own` false, run() computes them from elementary torch operations in fp32 (sums of log decays in fp64);
with `own` true it calls the package. exact() restates them in fp64, token by token and expert by expert.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# linear-attention heads: (key heads, value heads, key dim, value dim)
WIDE, EVEN, SMALL, ODD = (16, 32, 128, 128), (8, 8, 128, 128), (2, 4, 64, 64), (1, 3, 64, 128)


# ---- cases -------------------------------------------------------------------------------------------------

def delta(n_seq, n, dtype, heads=WIDE, **more):
    hk, hv, dk, dv = heads
    return {"kind": "delta", "n_seq": n_seq, "n": n, "dtype": dtype, "k_heads": hk, "v_heads": hv, "key_dim": dk,
            "val_dim": dv, "gated": False, "snap": False, **more}


def moe(n, dtype, experts, top_k, hidden, ffn, padded=0):
    return {"kind": "moe", "n": n, "dtype": dtype, "experts": experts, "top_k": top_k, "hidden": hidden, "ffn": ffn,
            "padded": padded}


def conv(n_seq, n, channels, taps, dtype, bias=False):
    return {"kind": "conv", "n_seq": n_seq, "n": n, "channels": channels, "taps": taps, "dtype": dtype, "bias": bias}


def route(n, experts, top_k, renorm, ties=False):
    return {"kind": "route", "n": n, "experts": experts, "top_k": top_k, "renorm": renorm, "ties": ties}


def listed():
    return [
        # a decode step's convolution over the q, k and v channels of a layer
        {"name": "conv_decode", **conv(1, 1, 8192, 4, "f32")},
        # the same channels over a prompt chunk
        {"name": "conv_prefill_4k", **conv(1, 4096, 8192, 4, "bf16")},
        # a decode step of one sequence: where launches and latency are all there is
        {"name": "delta_decode", **delta(1, 1, "f32", gated=True)},
        # speculative verify of a batch: one token and three drafts, a state kept after each for rollback
        {"name": "delta_verify_16x4", **delta(16, 4, "bf16", snap=True)},
        # a short prompt of a length that no tile divides, fp32 activations as the projections give them
        {"name": "delta_prompt_333", **delta(1, 333, "f32", gated=True)},
        # a chunk of a long prompt, bf16 activations
        {"name": "delta_prefill_4k", **delta(1, 4096, "bf16", gated=True)},
        # the router of a decode step
        {"name": "route_decode", **route(1, 128, 8, True)},
        # the router of a prompt chunk, with equal logits among a token's
        {"name": "route_4k", **route(4096, 512, 10, True, ties=True)},
        # a decode step's experts
        {"name": "moe_decode", **moe(1, "f32", 128, 8, 2048, 512)},
        # a small batch of requests with free places, about one token an expert
        {"name": "moe_batch_13", **moe(13, "bf16", 128, 8, 2048, 512, padded=3)},
        # a short prompt through fewer experts of an odd width
        {"name": "moe_prompt_500", **moe(500, "f32", 32, 4, 1024, 352)},
        # a chunk of a long prompt
        {"name": "moe_prefill_2k", **moe(2048, "bf16", 128, 8, 2048, 512)},
    ]


def spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = {}
    for c in listed():
        w, (b, f) = work(c), top.get(c["kind"], (0, 0))
        top[c["kind"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        kind, dtype = rng.choice(["conv", "delta", "delta", "delta", "route", "moe", "moe", "moe"]), rng.choice(["f32", "bf16"])
        if kind == "conv":
            n_seq = rng.choice([1, 1, spread(rng, 2, 64)])
            c = conv(n_seq, rng.choice([1, spread(rng, 2, 8192)]), 8 * spread(rng, 8, 1024), rng.choice([2, 3, 4, 4]),
                     dtype, rng.random() < 0.5)
        elif kind == "delta":
            few = rng.random() < 0.5
            c = delta(rng.choice([1, spread(rng, 1, 48 if few else 6)]), spread(rng, 1, 12) if few else spread(rng, 13, 6000),
                      dtype, rng.choice([WIDE, WIDE, WIDE, EVEN, SMALL, ODD]), gated=rng.random() < 0.5,
                      snap=few and rng.random() < 0.5)
        elif kind == "route":
            experts = spread(rng, 4, 512)
            c = route(spread(rng, 1, 8192), experts, rng.randint(1, min(16, experts)), rng.random() < 0.7, rng.random() < 0.5)
        else:
            experts, n = spread(rng, 4, 128), spread(rng, 1, 2048)
            c = moe(n, dtype, experts, rng.randint(1, min(8, experts)), 32 * spread(rng, 8, 64), 32 * spread(rng, 3, 24),
                    min(n - 1, rng.choice([0, 0, 1])))
        w, most = work(c), top[kind]
        # no drawn case costs more than the largest listed one of its kind
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and c not in ({k: v for k, v in x.items() if k != "name"} for x in listed()):
            return c


def work(c):
    n = c["n"]
    size = 2 if c.get("dtype") == "bf16" else 4
    if c["kind"] == "conv":
        rows = c["n_seq"] * n
        ch, taps = c["channels"], c["taps"]
        return {"bytes": 2 * rows * ch * size + 2 * 4 * c["n_seq"] * (taps - 1) * ch + 4 * ch * (taps + c["bias"]),
                "flops": rows * ch * (2 * taps + 4)}
    if c["kind"] == "delta":
        hk, hv, dk, dv, rows = c["k_heads"], c["v_heads"], c["key_dim"], c["val_dim"], c["n_seq"] * n
        state = 4 * c["n_seq"] * hv * dk * dv
        row = size * (2 * hk * dk + (3 if c["gated"] else 2) * hv * dv) + 8 * hv
        return {"bytes": rows * row + 2 * state + (n * state if c["snap"] else 0), "flops": 7 * rows * hv * dk * dv}
    if c["kind"] == "route":
        return {"bytes": n * (4 * c["experts"] + 8 * c["top_k"]), "flops": 4 * n * c["experts"]}
    pairs = (n - c["padded"]) * c["top_k"]
    # experts that at least one of the pairs reaches, were every expert as likely
    hit = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** (n - c["padded"]))
    weights = 3 * c["hidden"] * c["ffn"]
    return {"bytes": hit * weights * (1 + 4 / 32) + 2 * n * c["hidden"] * size + 8 * n * c["top_k"],
            "flops": pairs * 2 * weights}


# ---- inputs ------------------------------------------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c.get("dtype", "f32")]

    def normal(*shape, sd=1.0):
        return torch.randn(shape, generator=g, device=DEV) * sd

    def uniform(*shape, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(shape, generator=g, device=DEV)

    s, n = {"case": c}, c["n"]
    if c["kind"] == "conv":
        b, ch, k = c["n_seq"], c["channels"], c["taps"]
        s["x"] = normal(b, n, ch).to(dt)
        s["w"] = normal(ch, k, sd=k ** -0.5)
        s["bias"] = normal(ch, sd=0.2) if c["bias"] else None
        s["state"] = normal(b, k - 1, ch).to(dt).float()  # earlier rows of the same type
        s["y"] = torch.empty_like(s["x"])
    elif c["kind"] == "delta":
        b, hk, hv, dk, dv = c["n_seq"], c["k_heads"], c["v_heads"], c["key_dim"], c["val_dim"]
        # q, k and v are slices of one convolution's output rows
        rows = normal(b, n, 2 * hk * dk + hv * dv)
        rows = (rows * torch.sigmoid(rows)).to(dt)
        s["q"] = rows[..., :hk * dk].unflatten(-1, (hk, dk))
        s["k"] = rows[..., hk * dk:2 * hk * dk].unflatten(-1, (hk, dk))
        s["v"] = rows[..., 2 * hk * dk:].unflatten(-1, (hv, dv))
        s["a"], s["b"] = normal(b, n, hv), normal(b, n, hv)
        # heads that forget within a token beside heads that remember thousands
        s["a_coef"] = -torch.exp(uniform(hv, lo=math.log(1e-3), hi=math.log(8.0)))
        s["dt_bias"] = normal(hv, sd=0.5)
        s["state"] = normal(b, hv, dk, dv, sd=0.3)
        s["z"] = normal(b, n, hv, dv).to(dt) if c["gated"] else None
        s["gamma"] = 1 + normal(dv, sd=0.1) if c["gated"] else None
        s["snap"] = torch.empty((b, n, hv, dk, dv), device=DEV) if c["snap"] else None
        s["out"] = torch.empty((b, n, hv, dv), device=DEV, dtype=dt)
    elif c["kind"] == "route":
        s["logits"] = normal(n, c["experts"], sd=2.0)
        if c["ties"]:
            s["logits"] = (s["logits"] * 8).round() / 8
        s["ids"] = torch.empty((n, c["top_k"]), device=DEV, dtype=torch.int32)
        s["weights"] = torch.empty((n, c["top_k"]), device=DEV)
    else:
        e, k, h, f = c["experts"], c["top_k"], c["hidden"], c["ffn"]

        def q8(rows, cols):
            w = torch.randint(-127, 128, (e, rows, cols), generator=g, device=DEV, dtype=torch.int8)
            return w, uniform(e, rows, cols // 32, lo=0.5, hi=1.5) / (73 * cols ** 0.5)

        s["gate"], s["up"], s["down"] = q8(f, h), q8(f, h), q8(h, f)
        s["x"] = normal(n, h).to(dt)
        # some experts are likelier than others; no token goes to one expert twice
        score = normal(n, e) + normal(e, sd=0.5)
        top = torch.topk(score, k, dim=1)
        s["ids"] = top.indices.to(torch.int32)
        s["weights"] = torch.softmax(top.values, dim=1)
        if c["padded"]:
            s["ids"][n - c["padded"]:] = -1
        s["y"] = torch.empty_like(s["x"])
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


_context = []


def context():
    """The program's one context, made at its first call."""
    if not _context:
        _context.append(package().Attention(16, 2, 256, 64, max_ctx=8192, max_tokens=64, rms_eps=EPS))
    return _context[0]


def run(s):
    kind = s["case"]["kind"]
    if own:
        att = context()
        if kind == "conv":
            att.conv_silu(s["x"], s["w"], s["state"], s["y"], bias=s["bias"])
            return {"y": s["y"], "state": s["state"]}
        if kind == "delta":
            att.delta_rule(s["q"], s["k"], s["v"], s["a"], s["b"], s["state"], s["out"], a_coef=s["a_coef"],
                           dt_bias=s["dt_bias"], z=s["z"], gamma=s["gamma"], snap=s["snap"])
            return {"out": s["out"], "state": s["state"], "snap": s["snap"]}
        if kind == "route":
            att.moe_route(s["logits"], s["ids"], s["weights"], renorm=s["case"]["renorm"])
            return {"ids": s["ids"], "weights": s["weights"]}
        att.moe(s["x"], s["ids"], s["weights"], s["gate"], s["up"], s["down"], s["y"])
        return {"y": s["y"]}
    return {"conv": plain_conv, "delta": plain_delta, "route": plain_route, "moe": plain_moe}[kind](s)


def plain_conv(s):
    taps, n = s["w"].shape[1], s["x"].shape[1]
    x = torch.cat([s["state"], s["x"].float()], 1)
    y = (x.unfold(1, n, 1).transpose(2, 3) * s["w"].t()[:, None]).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"]
    s["state"].copy_(x[:, n:])
    return {"y": (y * torch.sigmoid(y)).to(s["x"].dtype), "state": s["state"]}


def inverse(a):
    """(I + a)^-1 of strictly lower triangular [..., c, c], c a power of two: blocks of s joined to blocks of 2 s."""
    c = a.shape[-1]
    t = torch.eye(c, device=a.device).expand_as(a).contiguous()
    s = 1
    while s < c:
        blocks = [m.view(*m.shape[:-2], c // (2 * s), 2 * s, c // (2 * s), 2 * s).diagonal(dim1=-4, dim2=-2) for m in (a, t)]
        low, inv = (m.movedim(-1, -3) for m in blocks)
        blocks[1][..., s:, :s, :] = -(inv[..., s:, s:] @ low[..., s:, :s] @ inv[..., :s, :s]).movedim(-3, -1)
        s *= 2
    return t


def plain_delta(s):
    b, n, hv, dv = s["v"].shape
    hk, dk = s["k"].shape[2:]
    # a chunk of 64 tokens at a time; one token where the state after each is kept
    c = 1 if s["snap"] is not None else min(64, 1 << (n - 1).bit_length())
    chunks = -(-n // c)

    def rows(x):  # [b, n, heads, d] -> [b, heads, chunks, c, d], zeros behind the last token
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, chunks * c - n))
        return x.unflatten(1, (chunks, c)).permute(0, 3, 1, 2, 4).contiguous()

    def unit(x):
        x = x.float()
        return (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)).repeat_interleave(hv // hk, dim=2)

    x = s["a"] + s["dt_bias"]
    g = rows((s["a_coef"] * (torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))))[..., None])[..., 0]
    beta = rows(torch.sigmoid(s["b"])[..., None])
    q, k, v = rows(unit(s["q"]) * dk ** -0.5), rows(unit(s["k"])), rows(s["v"])
    total = torch.cumsum(g.double(), -1)
    low = torch.ones(c, c, device=DEV, dtype=torch.bool).tril()
    decay = torch.exp(torch.where(low, total[..., :, None] - total[..., None, :], -math.inf).float())
    kt = k.transpose(-1, -2).contiguous()
    t = inverse((beta * (k @ kt) * decay).tril(-1))
    since, left = torch.exp(total.float())[..., None], torch.exp((total[..., -1:] - total).float())[..., None]
    u0, w, p = t @ (beta * v), t @ (beta * since * k), (q @ kt) * decay
    qs, kl, end = q * since, kt * left.transpose(-1, -2), torch.exp(total[..., -1].float())[..., None, None]
    state, out = s["state"], []
    for i in range(chunks):
        u = u0[:, :, i] - w[:, :, i] @ state
        out.append(qs[:, :, i] @ state + p[:, :, i] @ u)
        state.mul_(end[:, :, i]).add_(kl[:, :, i] @ u)
        if s["snap"] is not None:
            s["snap"][:, i] = state
    o = torch.stack(out, 2).flatten(2, 3)[:, :, :n].transpose(1, 2)
    if s["z"] is not None:
        z = s["z"].float()
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["gamma"] * z * torch.sigmoid(z)
    return {"out": o.to(s["v"].dtype), "state": state, "snap": s["snap"]}


def plain_route(s):
    top = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    p = torch.exp(top.values - top.values[:, :1])
    ids, w = top.indices[:, :s["case"]["top_k"]], p[:, :s["case"]["top_k"]]
    w = w / (w if s["case"]["renorm"] else p).sum(1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": w}


def widened(q, at=None):
    """fp32 weights of planar Q8_0 experts, all of them or those at given places."""
    w, sc = (q[0], q[1]) if at is None else (q[0][at], q[1][at])
    return (w.unflatten(-1, (-1, 32)).float() * sc[..., None]).flatten(-2)


def plain_moe(s):
    n, k = s["ids"].shape
    e = s["case"]["experts"]
    ids = s["ids"].long().flatten()
    there = (ids >= 0) & (ids < e)
    x = s["x"].float()
    if n * k <= e:  # each pair with its own expert's weights
        at = torch.where(there, ids, 0)
        rows = x.repeat_interleave(k, 0)[:, :, None]
        h = widened(s["gate"], at) @ rows
        h = h * torch.sigmoid(h) * (widened(s["up"], at) @ rows)
        pairs = (widened(s["down"], at) @ h)[:, :, 0]
    else:  # pairs by expert, each expert's padded to the fullest's
        order = torch.argsort(torch.where(there, ids, e), stable=True)
        count = torch.bincount(torch.where(there, ids, e), minlength=e + 1)
        place = torch.arange(n * k, device=DEV) - (torch.cumsum(count, 0) - count)[torch.where(there, ids, e)[order]]
        most = int(count[:e].max())
        slot = torch.full((n * k,), e * most, device=DEV).index_copy_(
            0, order, torch.where(there[order], ids[order] * most + place, e * most))
        rows = torch.zeros(e * most + 1, x.shape[1], device=DEV)
        rows[slot] = x.repeat_interleave(k, 0)
        rows = rows[:-1].view(e, most, -1)
        h = rows @ widened(s["gate"]).transpose(1, 2)
        h = h * torch.sigmoid(h) * (rows @ widened(s["up"]).transpose(1, 2))
        pairs = torch.nn.functional.pad((h @ widened(s["down"]).transpose(1, 2)).flatten(0, 1), (0, 0, 0, 1))[slot]
    pairs = torch.where(there[:, None], pairs, 0) * s["weights"].reshape(-1, 1)
    return {"y": pairs.view(n, k, -1).sum(1).to(s["x"].dtype)}


# ---- the definition in fp64 ----------------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if c["kind"] == "conv":
        seen = torch.cat([d["state"], d["x"]], 1)
        y = sum(seen[:, j:j + c["n"]] * d["w"][:, j] for j in range(c["taps"]))
        y = y if d["bias"] is None else y + d["bias"]
        return {"y": y / (1 + torch.exp(-y)), "state": seen[:, c["n"]:]}
    if c["kind"] == "delta":
        head = torch.arange(c["v_heads"], device=DEV) // (c["v_heads"] // c["k_heads"])
        state, out, kept = d["state"], [], []
        for t in range(c["n"]):
            q, k = (v[:, t] / torch.sqrt((v[:, t] ** 2).sum(-1, keepdim=True) + EPS) for v in (d["q"], d["k"]))
            q, k = q[:, head] / math.sqrt(c["key_dim"]), k[:, head]
            g = d["a_coef"] * torch.nn.functional.softplus(d["a"][:, t] + d["dt_bias"], threshold=60)
            state = state * torch.exp(g)[..., None, None]
            u = (d["v"][:, t] - (k[..., None] * state).sum(-2)) / (1 + torch.exp(-d["b"][:, t]))[..., None]
            state = state + k[..., None] * u[..., None, :]
            out.append((q[..., None] * state).sum(-2))
            if c["snap"]:
                kept.append(state)
        o = torch.stack(out, 1)
        if c["gated"]:
            o = o / torch.sqrt((o ** 2).mean(-1, keepdim=True) + EPS) * d["gamma"] * d["z"] / (1 + torch.exp(-d["z"]))
        return {"out": o, "state": state, "snap": torch.stack(kept, 1) if c["snap"] else None}
    if c["kind"] == "route":
        ids, w, left = [], [], d["logits"].clone()
        for _ in range(c["top_k"]):
            best = left.max(1, keepdim=True).values
            at = torch.where(left == best, torch.arange(c["experts"], device=DEV), c["experts"]).min(1).values
            ids.append(at)
            w.append(torch.gather(d["logits"], 1, at[:, None])[:, 0])
            left.scatter_(1, at[:, None], -math.inf)
        w = torch.exp(torch.stack(w, 1) - w[0][:, None])
        whole = w if c["renorm"] else torch.exp(d["logits"] - d["logits"].max(1, keepdim=True).values)
        return {"ids": torch.stack(ids, 1).to(torch.int32), "weights": w / whole.sum(1, keepdim=True)}
    y = torch.zeros(c["n"], c["hidden"], device=DEV, dtype=torch.float64)
    for e in range(c["experts"]):
        tok, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not len(tok):
            continue
        gate, up, down = ((s[m][0][e].double().unflatten(-1, (-1, 32)) * s[m][1][e].double()[..., None]).flatten(-2)
                          for m in ("gate", "up", "down"))
        h = d["x"][tok] @ gate.t()
        h = h / (1 + torch.exp(-h)) * (d["x"][tok] @ up.t())
        y.index_add_(0, tok, (h @ down.t()) * d["weights"][tok, j][:, None])
    return {"y": y}
