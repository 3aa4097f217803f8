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
