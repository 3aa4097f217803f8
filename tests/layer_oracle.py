"""64-bit restatements of the linear-attention and expert operators (CPU, token by token and pair by pair), and the
error bounds their tests use. Inputs are tensors as the operators take them; outputs are float64."""
import math

import torch

EPS32 = 2.0 ** -24  # half a step of float32, relative
HALF = {torch.float32: EPS32, torch.bfloat16: 2.0 ** -8}  # torch.finfo(t).eps / 2


def f64(x):
    return None if x is None else x.detach().cpu().double()


def conv(x, w, state, bias=None, lens=None):
    """(y [n_seq, n, C], state, snap [n_seq, n, taps - 1, C], bound on |y|'s sum of terms)."""
    x, w, state, bias = f64(x), f64(w), f64(state).clone(), f64(bias)
    b, n, c = x.shape
    taps = w.shape[1]
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    snap = torch.zeros(b, n, taps - 1, c, dtype=torch.float64)
    for s in range(b):
        for t in range(n if lens is None else min(max(int(lens[s]), 0), n)):
            win = torch.cat([state[s], x[s, t][None]])
            terms = win * w.t()
            pre = terms.sum(0) + (0 if bias is None else bias)
            mag[s, t] = terms.abs().sum(0) + (0 if bias is None else bias.abs())
            y[s, t] = pre / (1 + torch.exp(-pre))
            state[s] = win[1:]
            snap[s, t] = state[s]
    return y, state, snap, mag


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def delta(q, k, v, a, b, state, a_coef=None, dt_bias=None, z=None, gamma=None, lens=None, tiled=False, eps=1e-6):
    """(out before the gated norm and after it, state, snap, scale): scale [n_seq, v_heads, val_dim] is the largest
    2-norm that a column of the state, or the column's value, had on the way."""
    dk, hk = k.shape[-1], k.shape[2]
    q, k, v, a, b, S = f64(q), f64(k), f64(v), f64(a), f64(b), f64(state).clone()
    n_seq, n, hv, dv = v.shape
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + eps) / math.sqrt(dk)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + eps)
    head = torch.arange(hv) % hk if tiled else torch.arange(hv) // (hv // hk)
    q, k = q[:, :, head], k[:, :, head]
    if a_coef is not None:
        a = f64(a_coef) * softplus(a + f64(dt_bias))
        b = 1 / (1 + torch.exp(-b))
    out = torch.zeros(n_seq, n, hv, dv, dtype=torch.float64)
    snap = torch.zeros(n_seq, n, hv, dk, dv, dtype=torch.float64)
    scale = S.norm(dim=2)
    for s in range(n_seq):
        for t in range(n if lens is None else min(max(int(lens[s]), 0), n)):
            M = S[s] * torch.exp(a[s, t])[:, None, None]
            u = b[s, t][:, None] * (v[s, t] - (k[s, t][:, :, None] * M).sum(1))
            S[s] = M + k[s, t][:, :, None] * u[:, None, :]
            out[s, t] = (q[s, t][:, :, None] * S[s]).sum(1)
            snap[s, t] = S[s]
            scale[s] = torch.maximum(torch.maximum(scale[s], S[s].norm(dim=1)), v[s, t].abs())
    gated = out
    if z is not None:
        z = f64(z)
        gated = out / torch.sqrt((out * out).mean(-1, keepdim=True) + eps) * f64(gamma) * z / (1 + torch.exp(-z))
    return out, gated, S, snap, scale


# How far fp32 results may be from 64 bits as a 2-norm, relative: errors of independent roundings, each 0.41 of half a step
# in the mean square, add as squares. In the chunked delta rule at most 400 reach a value at its full size: the additions of
# its four products (key_dim and three times a chunk's 64) and some tens in norms, gates and scales.
CHUNK_LIMIT = 0.41 * math.sqrt(400) * EPS32


def remembering(normal, n_seq, n, hk, hv, dk, dv, dtype):
    """Inputs of the delta rule that keep most of their state (decays of 1% a token), so that every product of the chunked
    form counts in its results; normal(*shape): standard normal values."""
    q, k, v = (normal(n_seq, n, h, d).to(dtype) for h, d in ((hk, dk), (hk, dk), (hv, dv)))
    return dict(q=q, k=k, v=v, a=-torch.exp(normal(n_seq, n, hv)) * 0.01, b=torch.sigmoid(1 + normal(n_seq, n, hv)),
                state=normal(n_seq, hv, dk, dv))


def cut(x, parts):
    """x as the sum of that many bf16 parts, each what rounding leaves to the next."""
    out, left = torch.zeros_like(x), x
    for _ in range(parts):
        part = left.float().bfloat16().double()
        out, left = out + part, left - part
    return out


def delta_chunks(q, k, v, a, b, state, parts, eps=1e-6):
    """The delta rule (direct gates) in chunks of 64 tokens in 64 bits, the products' operands cut to bf16 parts (three, or
    parts[name]): (out, state). Names: kk and qk the rows in K K^T and Q K^T, k and s in K S, t and x in T X, q and qs in
    Q S, p and u in P U, kt and w in K^T W."""
    def op(x, name):
        return cut(x, parts.get(name, 3))

    q, k, v, a, b, S = f64(q), f64(k), f64(v), f64(a), f64(b), f64(state).clone()
    hk, dk, hv = k.shape[2], k.shape[3], v.shape[2]
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + eps) / math.sqrt(dk)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + eps)
    head, out = torch.arange(hv) // (hv // hk), []
    for t in range(0, v.shape[1], 64):
        Q, K, V = (x[:, t:t + 64].transpose(1, 2) for x in (q[:, :, head], k[:, :, head], v))
        G, B = a[:, t:t + 64].cumsum(1).transpose(1, 2), b[:, t:t + 64].transpose(1, 2)[..., None]
        D, since, last = torch.exp(G[..., :, None] - G[..., None, :]).tril(), torch.exp(G)[..., None], G[..., -1:]
        A = (B * D * (op(K, "kk") @ op(K, "kk").transpose(2, 3))).tril(-1)
        T, P = torch.linalg.inv(torch.eye(A.shape[-1], dtype=A.dtype) + A), D * (op(Q, "qk") @ op(K, "qk").transpose(2, 3))
        U = op(T, "t") @ op(B * (V - since * (op(K, "k") @ op(S, "s"))), "x")
        out.append((since * (op(Q, "q") @ op(S, "qs")) + op(P, "p") @ op(U, "u")).transpose(1, 2))
        S = torch.exp(last)[..., None] * S + op(K, "kt").transpose(2, 3) @ op(torch.exp(last - G)[..., None] * U, "w")
    return torch.cat(out, 1), S


def moe_limit(hidden, ffn):
    """As CHUNK_LIMIT, for the experts: the additions of a gate and an up value, those of a result, and some tens beside."""
    return 0.41 * math.sqrt(2 * hidden + ffn + 100) * EPS32


def apart(got, want):
    """The 2-norm of the difference, relative."""
    return float((f64(got) - want).norm() / want.norm())


def route(logits, top_k, renorm):
    """(ids, weights) by repeated maximum; -inf and NaN are no choice."""
    n, e = logits.shape
    x = torch.where(torch.isnan(logits.cpu()), torch.tensor(-math.inf), logits.cpu()).double()
    ids, w = torch.full((n, top_k), -1, dtype=torch.int32), torch.zeros(n, top_k, dtype=torch.float64)
    for t in range(n):
        row = x[t].clone()
        top = float(row.max())
        p = torch.tensor([0.0 if v == -math.inf else 1.0 if v == top else math.exp(v - top) for v in row.tolist()])
        for j in range(top_k):
            best = float(row.max())
            if best == -math.inf:
                break
            i = min(i for i in range(e) if float(row[i]) == best)
            ids[t, j], w[t, j], row[i] = i, p[i], -math.inf
        whole = float(w[t].sum() if renorm else p.double().sum())
        if whole:
            w[t] /= whole
    return ids, w


def widen(q):
    w, s = q[0].cpu().double(), q[1].cpu().double()
    return (w.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def moe(x, ids, weights, gate, up, down):
    """(y, bound): bound [n, hidden] is the sum of the magnitudes that the rounding errors of a row scale with."""
    x, ids, weights = f64(x), ids.cpu(), f64(weights)
    gate, up, down = widen(gate), widen(up), widen(down)
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < gate.shape[0]:
                continue
            g, u = gate[e] @ x[t], up[e] @ x[t]
            sig = 1 / (1 + torch.exp(-g))
            h = g * sig * u
            # |dh| <= |silu'| |u| |dg| + |silu(g)| |du|, with dg, du scaled by the sums of magnitudes; |silu'| < 1.1
            gm, um = gate[e].abs() @ x[t].abs(), up[e].abs() @ x[t].abs()
            y[t] += weights[t, j] * (down[e] @ h)
            mag[t] += weights[t, j].abs() * (down[e].abs() @ (1.1 * u.abs() * gm + (g * sig).abs() * um + 4 * h.abs()))
    return y, mag
