"""The linear-attention and expert operators on the GPU against 64-bit restatements (layer_oracle.py): the short
convolution, the gated delta rule (token by token and in chunks), the router, the experts, and a run of them with the
projections as a layer stack calls them. Bounds are worst-case rounding bounds, written where they are computed."""
import math

import pytest
import torch

import layer_oracle as lo
from layer_oracle import EPS32, HALF, f64

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def att(qw):
    a = qw.Attention(4, 1, 64, 16, max_ctx=256, max_tokens=64)
    yield a
    a.close()


def gen(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return lambda *shape, sd=1.0: torch.randn(shape, generator=g, device=DEV) * sd


def close(got, want, bound, what):
    got, want = f64(got), f64(want)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3e} "
                           f"at a bound of {float(torch.as_tensor(bound).max()):.3e}, first at {bad.nonzero()[0].tolist()}")


# ---- the convolution ---------------------------------------------------------------------------------------

def conv_bound(x, w, state, bias, lens, dtype):
    y, st, snap, mag = lo.conv(x, w, state, bias, lens)
    # the sum: a rounding a term and the bias; through silu's slope (< 1.1); e^-s: its argument's rounding; dtype
    return y, st, snap, 1.1 * (w.shape[1] + 2) * EPS32 * mag + (2 * mag + 16) * EPS32 * y.abs() + HALF[dtype] * y.abs() * 1.01 + 1e-37


@pytest.mark.parametrize("n_seq,n,ch,taps,dtype,bias", [
    (1, 1, 64, 4, F32, False), (1, 1, 8, 2, BF16, True), (2, 2, 72, 4, F32, True), (3, 3, 40, 3, BF16, False),
    (1, 16, 128, 4, F32, False), (2, 17, 1032, 4, BF16, True), (5, 33, 264, 3, F32, True), (1, 131, 2048, 2, BF16, False),
    (64, 1, 520, 4, BF16, False)])
def test_conv(att, n_seq, n, ch, taps, dtype, bias):
    r = gen(n_seq * 1000 + n)
    x, w, state = r(n_seq, n, ch).to(dtype), r(ch, taps), r(n_seq, taps - 1, ch)
    b = r(ch) if bias else None
    y, snap = torch.empty_like(x), torch.empty(n_seq, n, taps - 1, ch, device=DEV)
    want, st, sn, bound = conv_bound(x, w, state, b, None, dtype)
    s2, y2 = state.clone(), torch.empty_like(x)
    att.conv_silu(x, w, state, y, bias=b, snap=snap)
    att.conv_silu(x, w, s2, y2, bias=b)
    close(y, want, bound, "y")
    assert torch.equal(f64(state), st) and torch.equal(f64(snap), sn)  # rows are copied
    assert torch.equal(s2, state) and torch.equal(y2, y)


def test_conv_lens_strides_and_rows_left_alone(att):
    """Sequences of 0, 1, 2, 5, all and (clamped) more tokens; x and y column slices of wider rows; rows past a
    sequence's end, and the columns beside the slice, stay as they were; garbage in unused rows stays unused."""
    r = gen(7)
    n_seq, n, ch, taps = 7, 37, 72, 4
    lens = [0, 1, 2, 5, 37, 99, -4]
    wide, out = r(n_seq, n, 136), torch.full((n_seq, n, 88), 7.0, device=DEV)
    x, y = wide[..., 24:24 + ch], out[..., 8:8 + ch]
    for s, l in enumerate(lens):
        x[s, max(l, 0):] = float("nan")
    w, state = r(ch, taps), r(n_seq, taps - 1, ch)
    want, st, _, bound = conv_bound(torch.nan_to_num(x), w, state, None, lens, F32)
    att.conv_silu(x, w, state, y, lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert torch.equal(f64(state), st)
    for s, l in enumerate(lens):
        l = min(max(l, 0), n)
        close(y[s, :l], want[s, :l], bound[s, :l], f"y of sequence {s}")
        assert (y[s, l:] == 7).all()
    assert (out[..., :8] == 7).all() and (out[..., 8 + ch:] == 7).all()


def test_conv_chunks_join(att):
    """A prompt cut in two calls gives the bits of one call."""
    r = gen(8)
    x, w, state = r(1, 50, 64), r(64, 4), r(1, 3, 64)
    y, y2, s2 = torch.empty_like(x), torch.empty_like(x), state.clone()
    att.conv_silu(x, w, state, y)
    for a, b in ((0, 1), (1, 3), (3, 30), (30, 50)):
        att.conv_silu(x[:, a:b], w, s2, y2[:, a:b])
    assert torch.equal(y, y2) and torch.equal(state, s2)


def far_rows(n, width, stride, dtype, fill):
    """n rows at a stride that puts the last behind 2^32 bytes."""
    flat = torch.empty((n - 1) * stride + width, dtype=dtype, device=DEV)
    t = flat.as_strided((1, n, width), (n * stride, stride, 1))
    t.copy_(fill)
    return t


def test_conv_offsets_past_32_bits(att):
    r = gen(9)
    n, ch, stride = 6, 64, 1 << 28
    src = r(1, n, ch)
    x, y = far_rows(n, ch, stride, F32, src), far_rows(n, ch, stride, F32, torch.zeros_like(src))
    w, state = r(ch, 4), r(1, 3, ch)
    want, st, _, bound = conv_bound(src, w, state, None, None, F32)
    att.conv_silu(x, w, state, y)
    close(y, want, bound, "y")
    assert torch.equal(f64(state), st)


# ---- the gated delta rule ----------------------------------------------------------------------------------

def delta_inputs(seed, n_seq, n, hk, hv, dk, dv, dtype, coef=True, gated=False):
    r = gen(seed)
    rows = r(n_seq, n, 2 * hk * dk + 2 * hv * dv).to(dtype)  # q, k, v and z as slices of one buffer's rows
    q, k, v, z = rows.split([hk * dk, hk * dk, hv * dv, hv * dv], dim=2)
    d = dict(q=q.unflatten(2, (hk, dk)), k=k.unflatten(2, (hk, dk)), v=v.unflatten(2, (hv, dv)), a=r(n_seq, n, hv),
             b=r(n_seq, n, hv), state=r(n_seq, hv, dk, dv, sd=0.5))
    if coef:
        d.update(a_coef=-torch.exp(r(hv, sd=1.5)), dt_bias=r(hv))
    else:
        d.update(a=-torch.exp(d["a"]) * 0.3, b=torch.sigmoid(d["b"]))
    if gated:
        d.update(z=z.unflatten(2, (hv, dv)), gamma=1 + r(dv, sd=0.1))
    return d


def delta_run(att, d, snap=False, lens=None, tiled=False, fill=0.0, stream=None):
    state, out = d["state"].clone(), torch.full(d["v"].shape, fill, dtype=d["v"].dtype, device=DEV)
    kept = torch.full((*d["v"].shape[:3], *state.shape[2:]), fill, device=DEV) if snap else None
    att.delta_rule(**{**d, "state": state}, out=out, snap=kept, tiled=tiled, stream=stream,
                   lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV))
    return out, state, kept


def delta_check(att, d, snap=False, lens=None, tiled=False):
    """A token's step changes a column s of the state by products with vectors of 2-norm at most 1, each rounded some
    tens of times (normalized k: 10 roundings, S^T k: 12, u and the update: 10, decay: 4; in chunks three-part
    products, each part pair as a sum, and the chunk's inverse: 8 times as many), and no step enlarges what earlier ones
    left: after n tokens a column is off by at most 40 (n + 1) roundings (320) of the largest norm it, or its value,
    had. The output reads it through q, of norm 1 / sqrt(dk), twice (the state and k . q u)."""
    n, dk, dtype = d["v"].shape[1], d["k"].shape[3], d["v"].dtype
    oracle = {k: v for k, v in d.items()}
    o, gated, S, sn, scale = lo.delta(**oracle, lens=lens, tiled=tiled)
    out, state, kept = delta_run(att, d, snap, lens, tiled, fill=7.0)
    per = 40 if snap or n <= 16 else 320
    E = per * (n + 1) * EPS32 * scale[:, :, None, :]
    close(state, S, E, "state")
    Eo = (2 / math.sqrt(dk)) * E.permute(0, 2, 1, 3)
    if d.get("z") is not None:
        z, gamma = f64(d["z"]), f64(d["gamma"])
        rms = 1 / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-6)
        gate = rms * (gamma * z / (1 + torch.exp(-z))).abs()
        # through the norm: the element's own error, and the norm's, of rms(Eo), on the element
        Eo = 2 * gate * (Eo + o.abs() * rms * (Eo * Eo).mean(-1, keepdim=True).sqrt()) + (2 * z.abs() + 24) * EPS32 * gated.abs()
    bound = Eo + HALF[dtype] * gated.abs() * 1.01
    for s in range(d["v"].shape[0]):
        l = n if lens is None else min(max(lens[s], 0), n)
        close(out[s, :l], gated[s, :l], bound.expand_as(gated)[s, :l], f"out of sequence {s}")
        assert (out[s, l:] == 7).all()
        if snap:
            close(kept[s, :l], sn[s, :l], E[s], f"snap of sequence {s}")
            assert (kept[s, l:] == 7).all()
    return out, state


@pytest.mark.parametrize("n_seq,n,hk,hv,dk,dv,dtype,coef,gated,tiled", [
    (1, 1, 2, 4, 128, 128, F32, True, True, False), (3, 1, 1, 3, 64, 64, BF16, False, False, False),
    (2, 4, 2, 4, 128, 128, BF16, True, False, True), (1, 15, 1, 1, 64, 128, F32, True, True, False),
    (1, 16, 2, 2, 128, 64, F32, False, True, False), (1, 17, 2, 2, 128, 128, F32, True, False, False),
    (2, 33, 1, 2, 64, 64, BF16, True, True, False), (1, 63, 2, 4, 128, 128, F32, True, False, True),
    (1, 64, 1, 1, 128, 128, F32, True, True, False), (1, 65, 2, 2, 128, 128, BF16, True, True, False),
    (3, 77, 1, 3, 64, 128, F32, False, True, False), (2, 128, 2, 4, 128, 64, BF16, False, False, True),
    (1, 200, 1, 2, 128, 128, F32, True, True, False), (1, 333, 1, 1, 64, 64, F32, True, False, False)])
def test_delta(att, n_seq, n, hk, hv, dk, dv, dtype, coef, gated, tiled):
    delta_check(att, delta_inputs(n * 7 + n_seq, n_seq, n, hk, hv, dk, dv, dtype, coef, gated), tiled=tiled)


@pytest.mark.parametrize("n,dtype,gated", [(1, F32, True), (4, BF16, False), (19, F32, False)])
def test_delta_snapshots(att, n, dtype, gated):
    d = delta_inputs(50 + n, 2, n, 1, 2, 128, 128, dtype, True, gated)
    delta_check(att, d, snap=True)


@pytest.mark.parametrize("n,snap", [(9, True), (9, False), (150, False)])
def test_delta_lens(att, n, snap):
    """Ragged sequences (none, one, a chunk's edge, all, clamped ones); NaN in the rows that nothing may use."""
    lens = [0, 1, n, 64, n + 5, -1, 5, n - 1]
    d = delta_inputs(60 + n, len(lens), n, 1, 2, 64, 64, F32, True, True)
    clean = {k: v.clone() for k, v in d.items()}
    for s, l in enumerate(lens):
        for name in ("q", "k", "v", "z", "a", "b"):
            d[name][s, min(max(l, 0), n):] = float("nan")
            clean[name][s, min(max(l, 0), n):] = 0
    out, state, kept = delta_run(att, d, snap, lens, fill=7.0)
    delta_check(att, clean, snap, lens)
    out2, state2, kept2 = delta_run(att, clean, snap, lens, fill=7.0)
    assert torch.equal(out, out2) and torch.equal(state, state2)
    if snap:
        assert torch.equal(kept, kept2)


@pytest.mark.parametrize("n", [12, 130])
@pytest.mark.parametrize("case", ["same_keys", "forget", "remember", "beta_zero", "beta_one", "zero_rows", "huge", "reset"])
def test_delta_edges(att, case, n):
    d = delta_inputs(70 + n, 1, n, 1, 2, 128, 128, F32, False)
    if case == "same_keys":  # one key over and over, all of it rewritten each time
        d["k"][:] = d["k"][:, :1].clone()
        d["b"][:], d["a"][:] = 1.0, 0.0
    elif case == "forget":
        d["a"][:] = -40.0
    elif case == "remember":
        d["a"][:] = 0.0
    elif case == "beta_zero":
        d["b"][:] = 0.0
    elif case == "beta_one":
        d["b"][:] = 1.0
    elif case == "zero_rows":
        d["k"][:, ::3] = 0
        d["q"][:, ::5] = 0
        d["v"][:, ::2] = 0
    elif case == "huge":  # one token's value, then none like it
        d["v"][:, n // 2] *= 1e12
    else:  # a log decay of -inf starts afresh
        d["a"][:, n // 2] = -math.inf
    delta_check(att, d)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [12, 200])
def test_delta_token_that_is_not_finite(att, n, dtype):
    """A NaN value reaches its own sequence and head alone, and no token before it (in chunks: before its chunk)."""
    d = delta_inputs(90 + n, 2, n, 1, 2, 64, 64, dtype, True, True)
    bad = {k: v.clone() for k, v in d.items()}
    at = n - 3
    bad["v"][1, at, 0] = float("nan")
    out, state, _ = delta_run(att, d)
    out2, state2, _ = delta_run(att, bad)
    assert torch.equal(out[0], out2[0]) and torch.equal(state[0], state2[0])
    assert torch.equal(out[1, :, 1], out2[1, :, 1]) and torch.equal(state[1, 1], state2[1, 1])
    before = at if n < 64 else at // 64 * 64
    assert torch.equal(out[1, :before, 0], out2[1, :before, 0])
    assert torch.isnan(out2[1, at:, 0]).all() and torch.isnan(state2[1, 0]).all()


@pytest.mark.parametrize("gated", [False, True])
def test_delta_bf16_chunks_where_terms_cancel(att, gated):
    """bf16 outputs that are 2^-13 of their terms: q reads pairs of tokens whose keys are unit vectors and whose updates,
    fp32 values of 24 bits, cancel but for that (within a chunk and, through the state, from the one before). A term takes
    at most 24 roundings to fp32: beta v one, its key's and q's norms four each, the scales they enter four, decay,
    products and sums of parts the rest. Operands cut to 16 bits would be off by up to 2^-16 of a term, 2^-3 of an output."""
    n, dk, dv, hv = 100, 128, 64, 2
    d = delta_inputs(77, 1, n, 1, hv, dk, dv, BF16, False, gated)
    d["state"].zero_(), d["a"].zero_(), d["q"].zero_(), d["k"].zero_()
    g = torch.Generator().manual_seed(78)
    d["q"][0, 0, 0, 0] = 1
    for t in range(n):
        d["k"][0, t, 0, t] = 1
        if t:
            m = int(torch.randint((t + 1) // 2, (1,), generator=g))
            d["q"][0, t, 0, 2 * m:2 * m + 2] = 1
    d["v"][:] *= 512
    d["v"][:, 1::2] = -d["v"][:, ::2]
    d["b"][:] = 0.5 + 0.4 * torch.rand(1, n, hv, generator=g).to(DEV)
    d["b"][:, 1::2] = d["b"][:, ::2] * (1 - 2.0 ** -13)
    o, want, _, _, _ = lo.delta(**d)
    # every token's sum of magnitudes: the same with all values positive
    term = lo.delta(**{**d, "v": d["v"].abs()})[0]
    E = 24 * EPS32 * term
    if gated:
        z, gamma = f64(d["z"]), f64(d["gamma"])
        rms = 1 / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-6)
        gate = rms * (gamma * z / (1 + torch.exp(-z))).abs()
        E = 2 * gate * (E + o.abs() * rms * (E * E).mean(-1, keepdim=True).sqrt()) + (2 * z.abs() + 24) * EPS32 * want.abs()
    out, _, _ = delta_run(att, d)
    close(out, want, E + HALF[BF16] * want.abs() * 1.01, "out")
    assert float((o[0, 1:].abs() / term[0, 1:]).max()) < 2.0 ** -13  # the case is the one meant


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [12, 200])
@pytest.mark.parametrize("name", ["a", "b", "q", "k", "v", "a_coef", "dt_bias"])
def test_delta_nan_in_any_operand(att, name, n, dtype):
    """A NaN reaches every output and state that the definition computes from it: a gate's or value's its head from its
    token on, a key's the key head's value heads, a query's its token's outputs alone, a parameter's its head in every
    sequence; what it does not reach (in chunks: and earlier tokens of its chunk) has the bits of a clean call."""
    d = delta_inputs(190 + n, 2, n, 2, 4, 64, 64, dtype, True, True)
    bad, at = {k: v.clone() for k, v in d.items()}, n - 3
    seqs, rows, heads = [1], slice(at, n), [0]
    if name in ("a", "b"):
        bad[name][1, at, 0] = float("nan")
    elif name == "v":
        bad[name][1, at, 0, 5] = float("nan")
    elif name in ("q", "k"):
        bad[name][1, at, 0, 5] = float("nan")
        heads, rows = [0, 1], slice(at, at + 1) if name == "q" else rows
    else:
        bad[name][0] = float("nan")
        seqs, rows = [0, 1], slice(0, n)
    out, state, _ = delta_run(att, d)
    out2, state2, _ = delta_run(att, bad)
    reached = torch.zeros(2, n, 4, dtype=torch.bool, device=DEV)
    free = torch.ones_like(reached)
    first = rows.start if n < 64 else rows.start // 64 * 64
    for s in seqs:
        for h in heads:
            reached[s, rows, h] = True
            free[s, first if name != "q" else rows.start:rows.stop, h] = False
            if name != "q":
                # a value's NaN stays in its column of the state, and the gated norm spreads it over the output
                where = state2[s, h, :, 5] if name == "v" else state2[s, h]
                assert torch.isnan(where).all(), f"state of sequence {s}, head {h}"
    assert torch.isnan(out2[reached]).all()
    assert torch.equal(out2[free], out[free]) and torch.isfinite(out2[free]).all()
    kept = [(s, h) for s in range(2) for h in range(4) if name == "q" or not (s in seqs and h in heads)]
    assert all(torch.equal(state2[s, h], state[s, h]) for s, h in kept)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_seq,n,hk,hv,dk,dv", [(1, 333, 1, 2, 64, 64), (2, 65, 2, 2, 128, 128), (1, 200, 1, 1, 128, 64),
                                                 (1, 1000, 2, 4, 64, 128)])
def test_delta_chunks_of_fp32_accuracy(att, n_seq, n, hk, hv, dk, dv, dtype):
    """Beside the worst case: the 2-norm of the errors, within what independent roundings to fp32 make of it (any operand
    short of one of its three parts is beyond: test_layer_accuracy.py). A bf16 output is not looked at here."""
    d = lo.remembering(gen(500 + n), n_seq, n, hk, hv, dk, dv, dtype)
    want, _, S, _, _ = lo.delta(**d)
    out, state, _ = delta_run(att, d)
    errors = {"state": lo.apart(state, S), **({"out": lo.apart(out, want)} if dtype is F32 else {})}
    assert max(errors.values()) <= lo.CHUNK_LIMIT, errors


def test_delta_chunks_join(att):
    """A prompt in one call, in ragged calls of both forms, and token by token: states and outputs agree."""
    d = delta_inputs(80, 1, 150, 2, 4, 128, 128, F32, True, True)
    o, gated, S, _, scale = lo.delta(**d)
    for cuts in ([0, 150], [0, 1, 70, 134, 150], [0, 64, 128, 150], list(range(0, 40)) + [150]):
        state, out = d["state"].clone(), torch.empty_like(d["v"])
        for a, b in zip(cuts, cuts[1:]):
            part = {k: v[:, a:b] if k in ("q", "k", "v", "a", "b", "z") else v for k, v in d.items()}
            part["a"], part["b"] = part["a"].contiguous(), part["b"].contiguous()
            att.delta_rule(**{**part, "state": state}, out=out[:, a:b])
        close(state, S, 320 * 151 * EPS32 * scale[:, :, None, :], f"state of {cuts[:4]}")


def test_delta_segments_join(att):
    """More (chunk, head) pairs than are worked off at a time: the bits of the same sequences in calls of one segment."""
    d = delta_inputs(85, 32, 200, 16, 32, 64, 64, BF16, True, True)
    lens = [200 - 3 * i for i in range(32)]
    out, state, _ = delta_run(att, d, lens=lens)
    for s in range(0, 32, 8):
        part = {k: v[s:s + 8].contiguous() if k not in ("a_coef", "dt_bias", "gamma") else v for k, v in d.items()}
        o, st, _ = delta_run(att, part, lens=lens[s:s + 8])
        assert torch.equal(o, out[s:s + 8]) and torch.equal(st, state[s:s + 8])


def test_delta_same_bits_again(att):
    for n in (5, 300):
        d = delta_inputs(90 + n, 2, n, 2, 4, 128, 128, BF16, True, True)
        first = delta_run(att, d)
        for _ in range(3):
            again = delta_run(att, d)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("n", [6, 80])
def test_delta_offsets_past_32_bits(att, n):
    d = delta_inputs(95, 1, n, 1, 1, 64, 64, F32, True, True)
    far = dict(d)
    for name in ("q", "v", "z"):
        far[name] = far_rows(n, 64, (1 << 31) // n // 8 * 8, F32, d[name].flatten(2)).unflatten(2, (1, 64))
    out, state, _ = delta_run(att, d)
    s2, o2 = d["state"].clone(), far_rows(n, 64, (1 << 31) // n // 8 * 8, F32, torch.zeros(1, n, 64, device=DEV)).unflatten(2, (1, 64))
    att.delta_rule(**{**far, "state": s2}, out=o2)
    assert torch.equal(o2, out) and torch.equal(s2, state)


# ---- the router ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,experts,top_k,renorm", [
    (1, 1, 1, True), (1, 128, 8, True), (5, 7, 7, False), (3, 64, 64, True), (9, 65, 4, False), (6, 200, 10, True),
    (4, 512, 10, True), (3, 1000, 16, False), (2, 1024, 64, True), (5, 256, 8, False)])
def test_route(att, n, experts, top_k, renorm):
    r = gen(experts + n)
    logits = (r(n, experts + 3, sd=3.0) * 4).round() / 4  # many equal ones
    for x in (logits[:, :experts], logits[:, 2:experts + 2], logits[:, 1:experts + 1].contiguous()):  # strides, alignments
        ids, w = torch.empty(n, top_k, dtype=torch.int32, device=DEV), torch.empty(n, top_k, device=DEV)
        att.moe_route(x, ids, w, renorm=renorm)
        want_ids, want = lo.route(x, top_k, renorm)
        assert torch.equal(ids.cpu(), want_ids)
        # e^(l - max): the difference's rounding (|l - max| < 64) and the function's own; a sum of up to 1024; the division
        close(w, want, (64 + 4 + 24 + 2) * EPS32 * want + 1e-37, "weights")


def test_route_masked_rows(att):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 6, [nan] * 6, [-inf, 1, -inf, 2, nan, -inf], [inf, 0, inf, 1, 2, 3], [nan, 5, 5, -inf, 5, 5],
                      [-3e38, 3e38, 0, 0, 0, 0], [-0.0, 0.0, -0.0, 0.0, -1, -1]], device=DEV)
    for renorm in (True, False):
        ids, w = torch.empty(7, 3, dtype=torch.int32, device=DEV), torch.empty(7, 3, device=DEV)
        att.moe_route(x, ids, w, renorm=renorm)
        want_ids, want = lo.route(x, 3, renorm)
        assert torch.equal(ids.cpu(), want_ids), ids
        close(w, want, 100 * EPS32 * want + 1e-37, "weights")
    assert ids[0].tolist() == [-1, -1, -1] and ids[2].tolist() == [3, 1, -1] and ids[3].tolist() == [0, 2, 5]


# ---- the experts -------------------------------------------------------------------------------------------

def experts(seed, e, hidden, ffn):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def q8(rows, cols):
        return (torch.randint(-128, 128, (e, rows, cols), generator=g, device=DEV, dtype=torch.int8),
                (0.5 + torch.rand((e, rows, cols // 32), generator=g, device=DEV)) / (73 * cols ** 0.5))

    return q8(ffn, hidden), q8(ffn, hidden), q8(hidden, ffn)


def moe_check(att, x, ids, weights, q, what=""):
    y = torch.full_like(x, 7.0)
    att.moe(x, ids, weights, *q, y)
    want, mag = lo.moe(x, ids, weights, *q)
    # the longest sum (a rounding a 32-column block and some tens beside it) on the magnitudes, the split of the
    # activations (two parts: 2^-22) among them; dtype's rounding
    factor = (x.shape[1] / 32 + q[2][0].shape[2] / 32 + 48) * EPS32
    close(y, want, factor * mag + HALF[x.dtype] * want.abs() * 1.01, f"y {what}")
    return y


@pytest.mark.parametrize("n,e,k,hidden,ffn,dtype", [
    (1, 4, 2, 64, 32, F32), (1, 16, 4, 256, 96, BF16), (1, 3, 3, 2048, 512, F32), (2, 8, 2, 96, 64, F32),
    (3, 5, 5, 32, 32, BF16), (7, 16, 4, 288, 160, F32), (13, 64, 8, 512, 128, BF16), (20, 2, 1, 128, 352, F32),
    (33, 4, 2, 160, 96, BF16), (64, 8, 3, 256, 64, F32), (100, 1, 1, 128, 128, BF16), (150, 6, 4, 320, 224, F32),
    (257, 3, 2, 544, 96, BF16), (300, 40, 2, 128, 160, F32), (400, 40, 2, 160, 96, BF16), (1000, 4, 2, 96, 32, F32),
    (700, 5, 3, 288, 352, BF16), (513, 9, 2, 1056, 64, F32)])
def test_moe(att, n, e, k, hidden, ffn, dtype):
    r, q = gen(n * 3 + e), experts(n, e, hidden, ffn)
    x = r(n, hidden).to(dtype)
    top = torch.topk(r(n, e) + r(e), k, dim=1)
    moe_check(att, x, top.indices.to(torch.int32), torch.softmax(top.values, 1), q)


@pytest.mark.parametrize("n,e,k,hidden,ffn", [(1, 4, 2, 1056, 352), (200, 3, 2, 1056, 352), (700, 5, 3, 288, 352),
                                              (300, 40, 2, 128, 160)])
def test_moe_of_fp32_accuracy(att, n, e, k, hidden, ffn):
    """Beside the worst case: the 2-norm of the errors, in both forms and both heights of tiles (activations short of their
    second part are beyond it: test_layer_accuracy.py)."""
    r, q = gen(n * 5 + e), experts(n, e, hidden, ffn)
    x, w = r(n, hidden), r(n, k)
    ids = torch.topk(r(n, e), k, dim=1).indices.to(torch.int32)
    y = torch.empty_like(x)
    att.moe(x, ids, w, *q, y)
    error = lo.apart(y, lo.moe(x, ids, w, *q)[0])
    assert error <= lo.moe_limit(hidden, ffn)


@pytest.mark.parametrize("n", [1, 6, 40, 200])
def test_moe_skipped_and_repeated_ids(att, n):
    """Ids outside the experts (free places, whole rows and single ones), one expert twice in a row, every token to one
    expert, negative and zero weights; no id at all gives rows of zeros."""
    e, k, hidden, ffn = 5, 4, 128, 96
    r, q = gen(n), experts(3, e, hidden, ffn)
    x, w = r(n, hidden), r(n, k)
    w[:, 1] = 0
    g = torch.Generator(device=DEV).manual_seed(n)
    ids = torch.randint(-2, e + 2, (n, k), generator=g, device=DEV, dtype=torch.int32)
    ids[0] = torch.tensor([2, 2, -1, 1 << 30], device=DEV)
    moe_check(att, x, ids, w, q, "mixed")
    moe_check(att, x, torch.full_like(ids, 3), w, q, "one expert")
    y = torch.full_like(x, 7.0)
    att.moe(x, torch.full_like(ids, -1), w, *q, y)
    assert (y == 0).all()


@pytest.mark.parametrize("n", [1, 50, 300])
def test_moe_rows_of_many_magnitudes(att, n):
    """Rows far from one another's size, values far from their row's largest, zero rows: each row is held to its own
    magnitude (in 64 bits, beside the largest finite values too far for fp32 products)."""
    r, q = gen(n + 1), experts(4, 3, 256, 64)
    x = r(n, 256) * torch.exp(r(n, 256, sd=3.0)) * 10.0 ** r(n, 1, sd=2.0).round()
    x[n // 2] = 0
    ids = torch.arange(2 * n, device=DEV, dtype=torch.int32).view(n, 2) % 3
    y = moe_check(att, x, ids, r(n, 2), q)
    assert (y[n // 2] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [4, 300, 700])
@pytest.mark.parametrize("power", [10, 28, 34])
def test_moe_values_beside_one_far_larger(att, n, dtype, power):
    """Rows with one value 2^power that no weight reads (its columns are zeros), so that only what the operands keep of the
    others shows: all of them by pairs; grouped each to 2^-23 of itself or 2^-39 of the row's largest. The same for h, one
    of whose values the down product does not read."""
    e, hidden, ffn = 3, 128, 96
    r, (gate, up, down) = gen(n + power), experts(12, e, hidden, ffn)
    gate[0][:, :, 5], up[0][:, :, 5] = 0, 0
    x, ids, w = r(n, hidden).to(dtype), torch.arange(2 * n, device=DEV, dtype=torch.int32).view(n, 2) % e, r(n, 2)
    x[:, 5] = 2.0 ** power
    gate[0][:, 7], up[0][:, 7], down[0][:, :, 7] = 127, 127, 0  # h's value 7 is large
    gate[1][:, 7], up[1][:, 7] = 8.0, 8.0
    y = torch.empty_like(x)
    att.moe(x, ids, w, gate, up, down, y)
    want, mag = lo.moe(x, ids, w, gate, up, down)
    # what the split leaves of x and h, through the same products
    G, U, D = (lo.widen(m) for m in (gate, up, down))
    G[:, 7], U[:, 7] = 0, 0  # (not read by the down product)
    kept = torch.zeros_like(want)
    dx = 2.0 ** -39 * 2.0 ** power * torch.ones(hidden, dtype=torch.float64)
    for t in range(n):
        for j in range(2):
            i, xt = int(ids[t, j]), f64(x[t])
            g, u = G[i] @ xt, U[i] @ xt
            s = 1 / (1 + torch.exp(-g))
            full = (lo.widen(gate)[i][7] @ xt, lo.widen(up)[i][7] @ xt)
            h7 = full[0] / (1 + torch.exp(-full[0])) * full[1]
            dh = 1.1 * u.abs() * (G[i].abs() @ dx) + (g * s).abs() * (U[i].abs() @ dx) + 2.0 ** -39 * max(h7.abs(), (g * s * u).abs().max())
            # (second order: the two errors of g and u meet)
            kept[t] += f64(w[t, j]).abs() * (D[i].abs() @ (dh + 1.1 * (G[i].abs() @ dx) * (U[i].abs() @ dx)))
    # (mag with |x|'s large value read by zeros, h's by zeros: neither counts)
    factor = (hidden / 32 + ffn / 32 + 48) * EPS32
    close(y, want, factor * mag + (0 if n == 4 else 1) * kept + HALF[dtype] * want.abs() * 1.01, "y")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 40, 300])
def test_moe_rows_that_are_not_finite(att, n, dtype):
    """Infinities and NaN in a token's row reach its own row of y alone; a NaN weight of a free place reaches nothing."""
    q, r = experts(9, 3, 256, 64), gen(n + 5)
    x, w = r(n, 256).to(dtype), r(n, 2)
    ids = torch.arange(2 * n, device=DEV, dtype=torch.int32).view(n, 2) % 3
    ids[3, 1], w[3, 1] = -1, float("nan")
    bad = x.clone()
    bad[0, 17], bad[2, 255], bad[n - 1] = float("nan"), float("inf"), float("-inf")
    y, y2 = torch.empty_like(x), torch.empty_like(x)
    att.moe(x, ids, w, *q, y)
    att.moe(bad, ids, w, *q, y2)
    rows = torch.ones(n, dtype=torch.bool, device=DEV)
    rows[[0, 2, n - 1]] = False
    assert torch.isfinite(y).all() and torch.equal(y[rows], y2[rows])
    assert not torch.isfinite(y2[~rows]).any()


def test_moe_strides_offsets_and_neighbours(att):
    """x and y as column slices, and as rows behind 2^32 bytes; columns beside the slice stay as they were."""
    q, r = experts(5, 4, 64, 96), gen(11)
    for n in (2, 40, 900):
        ids, w = torch.arange(n * 2, device=DEV, dtype=torch.int32).view(n, 2) % 4, r(n, 2)
        wide, out = r(n, 136), torch.full((n, 88), 7.0, device=DEV)
        x, y = wide[:, 8:72], out[:, 16:80]
        dense, far = torch.empty(n, 64, device=DEV), far_rows(n, 64, (1 << 31) // (n - 1) // 8 * 8, F32, x[None])[0]
        far_y = far_rows(n, 64, (1 << 31) // (n - 1) // 8 * 8, F32, torch.zeros(1, n, 64, device=DEV))[0]
        att.moe(x.contiguous(), ids, w, *q, dense)
        att.moe(x, ids, w, *q, y)
        att.moe(far, ids, w, *q, far_y)
        assert torch.equal(dense, y) and torch.equal(dense, far_y)
        assert (out[:, :16] == 7).all() and (out[:, 80:] == 7).all()


def test_moe_weights_past_32_bits(att):
    """An expert behind the first 4 GiB of the weights (and of the scales' elements) is read where it lies."""
    e, hidden, ffn = 1024, 2048, 2560
    small = experts(6, 2, hidden, ffn)
    q = [(torch.empty(e, *w.shape[1:], dtype=torch.int8, device=DEV), torch.empty(e, *s.shape[1:], device=DEV)) for w, s in small]
    for (w, s), (w2, s2) in zip(q, small):
        w[1023], s[1023], w[900], s[900] = w2[0], s2[0], w2[1], s2[1]
    r = gen(12)
    for n in (1, 40, 1300):
        x, ids, wt = r(n, hidden), torch.tensor([[1023, 900]], dtype=torch.int32, device=DEV).repeat(n, 1), r(n, 2)
        y, y2 = torch.empty_like(x), torch.empty_like(x)
        att.moe(x, ids, wt, *q, y)
        att.moe(x, (ids == 900).int(), wt, *small, y2)
        # the same pairs in the same order, whatever the number of experts chose as the form
        close(y, y2, 1e-5 * float(y2.abs().max()), f"n = {n}")


def test_moe_segments_join(att):
    """More pairs than are worked off at a time: the bits of the same rows in calls of one segment."""
    n, k, e = 20000, 4, 3
    q, r = experts(7, e, 64, 32), gen(14)
    g = torch.Generator(device=DEV).manual_seed(15)
    x, w = r(n, 64), r(n, k)
    ids = torch.randint(-1, e + 1, (n, k), generator=g, device=DEV, dtype=torch.int32)
    y, parts = torch.empty_like(x), torch.empty_like(x)
    att.moe(x, ids, w, *q, y)
    for a, b in ((0, 9000), (9000, n)):  # (both grouped: the form by pairs sums in another order)
        att.moe(x[a:b], ids[a:b], w[a:b], *q, parts[a:b])
    assert torch.equal(y, parts)
    want, mag = lo.moe(x[::499], ids[::499], w[::499], *q)
    close(y[::499], want, (64 / 32 + 32 / 32 + 48) * EPS32 * mag + EPS32 * want.abs(), "y")


def test_moe_same_bits_again(att):
    q, r = experts(8, 16, 512, 128), gen(13)
    for n, dtype in ((1, F32), (30, BF16), (400, F32)):
        x = r(n, 512).to(dtype)
        top = torch.topk(r(n, 16), 4, dim=1)
        ids, w, y = top.indices.int(), torch.softmax(top.values, 1), torch.empty_like(x)
        att.moe(x, ids, w, *q, y)
        first = y.clone()
        for _ in range(3):
            att.moe(x, ids, w, *q, y)
            assert torch.equal(y, first)


# ---- together, on streams and in graphs -----------------------------------------------------------------------

class Layer:
    """A linear-attention layer and an expert layer over fp32 rows of 256: qkv and z projections, convolution, delta
    rule with the gated norm, output projection; router projection, router, experts; residual sums."""
    H, HK, HV, D, E, K, F = 256, 1, 2, 64, 8, 2, 96

    def __init__(self, att, seed=20, n_seq=1):
        r, self.att = gen(seed), att
        self.qkv, self.zab = (2 * self.HK + self.HV) * self.D, self.HV * self.D + 2 * self.HV
        self.w_in, self.w_z = r(self.qkv, self.H, sd=1 / 16), r(self.zab, self.H, sd=1 / 16)
        self.w_out, self.w_r = r(self.H, self.HV * self.D, sd=1 / 11), r(self.E, self.H, sd=1 / 8)
        self.w_conv, self.a_coef, self.dt = r(self.qkv, 4, sd=0.5), -torch.exp(r(self.HV)), r(self.HV)
        self.gamma, self.q = 1 + r(self.D, sd=0.1), experts(seed, self.E, self.H, self.F)
        self.n_seq = n_seq
        self.conv = torch.zeros(n_seq, 3, self.qkv, device=DEV)
        self.state = torch.zeros(n_seq, self.HV, self.D, self.D, device=DEV)

    def buffers(self, n):
        rows = self.n_seq * n
        e = lambda *s, dtype=F32: torch.empty(s, device=DEV, dtype=dtype)
        ws = max(1, self.ws_bytes(n))
        return dict(qkv=e(rows, self.qkv), zab=e(rows, self.zab), mixed=e(self.n_seq, n, self.qkv), o=e(self.n_seq, n, self.HV, self.D),
                    proj=e(rows, self.H), logits=e(rows, self.E), ids=e(rows, self.K, dtype=torch.int32), w=e(rows, self.K),
                    y=e(rows, self.H), a=e(self.n_seq, n, self.HV), b=e(self.n_seq, n, self.HV), out=e(rows, self.H),
                    x1=e(rows, self.H), z=e(self.n_seq, n, self.HV, self.D), ws=e(ws, dtype=torch.uint8))

    def ws_bytes(self, n):
        import common
        qw = common.load_package()
        return max(qw.delta_workspace(self.n_seq, n, self.HK, self.HV, self.D, self.D, F32, True),
                   qw.moe_workspace(self.E, self.H, self.F, F32, self.n_seq * n, self.K))

    def forward(self, x, n, t, stream=None):
        """x [n_seq * n, H] -> t["out"], in t's buffers (no allocation)."""
        att, hk, hv, d = self.att, self.HK, self.HV, self.D
        att.mat_multi(x, [(t["qkv"], self.w_in, None), (t["zab"], self.w_z, None)], stream=stream)
        t["z"].copy_(t["zab"][:, :hv * d].view(self.n_seq, n, hv, d))
        t["a"].copy_(t["zab"][:, hv * d:hv * d + hv].view(self.n_seq, n, hv))
        t["b"].copy_(t["zab"][:, hv * d + hv:].view(self.n_seq, n, hv))
        att.conv_silu(t["qkv"].view(self.n_seq, n, -1), self.w_conv, self.conv, t["mixed"], stream=stream)
        q, k, v = t["mixed"].split([hk * d, hk * d, hv * d], dim=2)
        att.delta_rule(q.unflatten(2, (hk, d)), k.unflatten(2, (hk, d)), v.unflatten(2, (hv, d)), t["a"], t["b"], self.state,
                       t["o"], a_coef=self.a_coef, dt_bias=self.dt, z=t["z"], gamma=self.gamma, workspace=t["ws"], stream=stream)
        att.mat(t["o"].view(-1, hv * d), t["proj"], self.w_out, stream=stream)
        torch.add(x, t["proj"], out=t["x1"])
        att.mat(t["x1"], t["logits"], self.w_r, stream=stream)
        att.moe_route(t["logits"], t["ids"], t["w"], stream=stream)
        att.moe(t["x1"], t["ids"], t["w"], *self.q, t["y"], workspace=t["ws"], stream=stream)
        torch.add(t["x1"], t["y"], out=t["out"])
        return t["out"]

    def oracle(self, x, ids):
        """The same in 64 bits from zero states; `ids`: the experts that the GPU chose (a near tie may fall either way)."""
        hk, hv, d, x = self.HK, self.HV, self.D, f64(x)
        n = x.shape[0] // self.n_seq
        qkv, zab = x @ f64(self.w_in).t(), x @ f64(self.w_z).t()
        mixed = lo.conv(qkv.view(self.n_seq, n, -1), self.w_conv, torch.zeros_like(self.conv))[0]
        q, k, v = mixed.split([hk * d, hk * d, hv * d], dim=2)
        z, a, b = zab.view(self.n_seq, n, -1).split([hv * d, hv, hv], dim=2)
        o = lo.delta(q.unflatten(2, (hk, d)), k.unflatten(2, (hk, d)), v.unflatten(2, (hv, d)), a, b, torch.zeros_like(self.state),
                     self.a_coef, self.dt, z.unflatten(2, (hv, d)), self.gamma)[1]
        x1 = x + o.reshape(-1, hv * d) @ f64(self.w_out).t()
        logits = x1 @ f64(self.w_r).t()
        w = torch.softmax(torch.gather(logits, 1, ids.cpu().long()), 1)
        best = torch.sort(logits, 1, descending=True).values[:, :self.K]
        assert (torch.gather(logits, 1, ids.cpu().long()) >= best - 1e-3).all()
        return x1 + lo.moe(x1, ids, w, *self.q)[0]


@pytest.mark.parametrize("n_seq,cuts", [(1, [0, 90, 91, 92, 96]), (2, [0, 3, 4, 40])])
def test_layers_together(att, n_seq, cuts):
    """A prompt chunk, then decode and verify-sized calls, through both layers, against 64 bits: rows agree to 1e-4 of
    their size (a dozen chained operators of fp32 accuracy, each within some hundred roundings of 6e-8)."""
    L, n = Layer(att, n_seq=n_seq), cuts[-1]
    x = gen(30)(n_seq, n, L.H)
    got, ids = torch.empty_like(x), torch.empty(n_seq, n, L.K, dtype=torch.int32, device=DEV)
    for a, b in zip(cuts, cuts[1:]):
        t = L.buffers(b - a)
        got[:, a:b] = L.forward(x[:, a:b].reshape(-1, L.H), b - a, t).view(n_seq, b - a, -1)
        ids[:, a:b] = t["ids"].view(n_seq, b - a, -1)
    want = L.oracle(x.view(-1, L.H), ids.view(-1, L.K))
    err = (f64(got.view(-1, L.H)) - want).norm(dim=1) / want.norm(dim=1)
    assert float(err.max()) < 1e-4


@pytest.mark.parametrize("n", [1, 4, 100])
def test_layers_in_a_graph(att, n):
    """Both layers captured and replayed several times, eager work on the same context between the replays: each replay's
    outputs and states have the bits of the same eager steps."""
    L, E = Layer(att), Layer(att)
    t, te = L.buffers(n), E.buffers(n)
    xs = [gen(40 + i)(n, L.H) for i in range(4)]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L.forward(x, n, t)  # (modules load outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    L.conv.zero_(), L.state.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.forward(x, n, t)
    for i in range(4):
        x.copy_(xs[i])
        g.replay()
        want = E.forward(xs[i], n, te)
        torch.cuda.synchronize()
        assert torch.equal(t["out"], want), f"replay {i}"
        assert torch.equal(L.state, E.state) and torch.equal(L.conv, E.conv)


def test_two_streams_at_once(att):
    """Calls on two streams with their own states and workspaces, interleaved, give the bits of calls alone; the
    operators run on the stream they are given."""
    outs = []
    for together in (False, True):
        layers = [Layer(att, seed=21), Layer(att, seed=22)]
        ts = [L.buffers(70) for L in layers]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for i in range(3):
            for L, t, s in zip(layers, ts, streams):
                with torch.cuda.stream(s):
                    L.forward(gen(50 + i)(70, L.H), 70, t, stream=s if together else None)
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        outs.append([t["out"].clone() for t in ts] + [L.state.clone() for L in layers])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_workspace_for_smaller_calls(att, qw, dtype):
    """A workspace for the largest call serves every smaller one (fewer sequences can need more than the largest): the
    bits of calls with workspaces of their own, whatever bytes the last call left in it."""
    hk, hv, d = 16, 32, 64
    size = qw.delta_workspace(40, 130, hk, hv, d, d, dtype, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    for n_seq, n in ((40, 130), (33, 130), (32, 130), (3, 130), (1, 130), (1, 40), (40, 40), (7, 19)):
        i = delta_inputs(300 + n_seq, n_seq, n, hk, hv, d, d, dtype, True, True)
        out, state, _ = delta_run(att, i)
        s2, o2 = i["state"].clone(), torch.empty_like(out)
        att.delta_rule(**{**i, "state": s2}, out=o2, workspace=ws)
        assert torch.equal(out, o2) and torch.equal(state, s2), (n_seq, n)
    q, e, k = experts(10, 8, 128, 96), 8, 2
    ws = torch.full((qw.moe_workspace(e, 128, 96, dtype, 700, k),), 255, dtype=torch.uint8, device=DEV)
    for n in (700, 300, 31, 5, 1):
        r = gen(n)
        x, ids, w = r(n, 128).to(dtype), torch.arange(n * k, device=DEV, dtype=torch.int32).view(n, k) % e, r(n, k)
        y, y2 = torch.empty_like(x), torch.empty_like(x)
        att.moe(x, ids, w, *q, y)
        att.moe(x, ids, w, *q, y2, workspace=ws)
        assert torch.equal(y, y2), n


def test_library_refuses_on_the_gpu(att, qw):
    """The library's own checks behind the mirror's: an error with its text, nothing launched."""
    z = lambda *s, dtype=F32: torch.zeros(s, device=DEV, dtype=dtype)
    with pytest.raises(qw.QwattnError, match="channels 12"):
        att.conv_silu(z(1, 2, 12), z(12, 4), z(1, 3, 12), z(1, 2, 12))
    x = z(1, 2, 16)
    with pytest.raises(qw.QwattnError, match="x and y overlap"):
        att.conv_silu(x, z(16, 4), z(1, 3, 16), x)
    v = z(1, 2, 3, 64)
    with pytest.raises(qw.QwattnError, match="v_heads 3"):
        att.delta_rule(z(1, 2, 2, 64), z(1, 2, 2, 64), v, z(1, 2, 3), z(1, 2, 3), z(1, 3, 64, 64), z(1, 2, 3, 64))
    with pytest.raises(qw.QwattnError, match="come together"):
        att.delta_rule(z(1, 2, 1, 64), z(1, 2, 1, 64), v, z(1, 2, 3), z(1, 2, 3), z(1, 3, 64, 64), z(1, 2, 3, 64), dt_bias=z(3))
    with pytest.raises(qw.QwattnError, match="top_k 9"):
        att.moe_route(z(2, 8), z(2, 9, dtype=torch.int32), z(2, 9))
    q = experts(1, 2, 64, 32)
    with pytest.raises(qw.QwattnError, match="workspace"):
        att.moe(z(2, 64), z(2, 1, dtype=torch.int32), z(2, 1), *q, z(2, 64), workspace=z(8, dtype=torch.uint8))
