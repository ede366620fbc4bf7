"""Plain 64-bit implementations of the routing from logits and of the 8-bit
block products, on the CPU (numpy), written from their definitions."""
from __future__ import annotations

import numpy as np

E4M3_MAX = 448.0
LEAST = 2.0 ** -100


# ---- routing ------------------------------------------------------------------


def route_scores(logits, score):
    """s (R, E) float64, 0 for experts that take no part."""
    l = np.asarray(logits, np.float64)
    live = l > -np.inf  # (a NaN is not)
    s = np.zeros_like(l)
    for r in range(l.shape[0]):
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                s[r, live[r]] = 1.0 / (1.0 + np.exp(-l[r, live[r]]))
        elif live[r].any():
            v = l[r, live[r]]
            m = v.max()
            with np.errstate(invalid="ignore"):
                e = np.where(v == m, 1.0, np.exp(v - m))
            s[r, live[r]] = e / e.sum()
    return s, live


def route(logits, k, bias=None, score="softmax", n_groups=1, top_groups=None, group_score="max", renormalize=True,
          scale=1.0):
    """(inds (R, k) int, gates (R, k) float64)."""
    l = np.asarray(logits, np.float64)
    R, E = l.shape
    top_groups = n_groups if top_groups is None else top_groups
    s, live = route_scores(l, score)
    b = np.zeros(E) if bias is None else np.asarray(bias, np.float64)
    alive = live & (b > -np.inf)
    value = s + np.where(b > -np.inf, b, 0.0)
    rank = l if bias is None else value
    inds = np.zeros((R, k), np.int64)
    gates = np.zeros((R, k))
    S = E // n_groups
    for r in range(R):
        order = range(E)
        if n_groups > 1:
            gs = []
            for g in range(n_groups):
                mine = [e for e in range(g * S, (g + 1) * S) if alive[r, e]]
                if not mine:
                    gs.append(-np.inf)
                elif group_score == "max":
                    gs.append(max(rank[r, e] for e in mine))
                else:
                    gs.append(sum(sorted((value[r, e] for e in mine), reverse=True)[:2]))
            best = sorted(range(n_groups), key=lambda g: (-gs[g], g))[:top_groups]
            order = [e for g in sorted(best) for e in range(g * S, (g + 1) * S)]
        chosen = sorted(order, key=lambda e: (0, -rank[r, e], e) if alive[r, e] else (1, 0.0, e))[:k]
        inds[r] = chosen
        w = np.array([s[r, e] if alive[r, e] else 0.0 for e in chosen])
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else w
        gates[r] = scale * w
    return inds, gates


def route_backward(logits, inds, gates, d_gates, score="softmax", renormalize=True, scale=1.0):
    """d_logits (R, E) float64 of fixed inds; slots whose gate is 0 took no part."""
    l = np.asarray(logits, np.float64)
    R, E = l.shape
    s, _ = route_scores(l, score)
    out = np.zeros((R, E))
    for r in range(R):
        ds = np.zeros(E)
        on = [j for j in range(inds.shape[1]) if gates[r, j] != 0]
        U = sum(s[r, inds[r, j]] for j in on)
        for j in on:
            d = scale * d_gates[r, j]
            if renormalize:
                d = (d - sum(scale * d_gates[r, i] * s[r, inds[r, i]] for i in on) / U) / U
            ds[inds[r, j]] += d
        if score == "sigmoid":
            out[r] = ds * s[r] * (1.0 - s[r])
        else:
            out[r] = s[r] * (ds - (ds * s[r]).sum())
    return out


# ---- 8-bit blocks ---------------------------------------------------------------


def e4m3(v):
    """To the nearest e4m3 value, ties to even (NaN stays; |v| < 464)."""
    v = np.asarray(v, np.float64)
    _, e = np.frexp(v)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(v / step) * step


def _round_block(b):
    """(values q, scale) of one block (fp32 values)."""
    b = np.asarray(b, np.float32)
    a = np.maximum(np.abs(b).max() if b.size else np.float32(0), np.float32(LEAST)).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        up, down = np.float32(E4M3_MAX) / a, a / np.float32(E4M3_MAX)
        return e4m3((b * up).astype(np.float32)), np.float64(down)


def quantize_rows(x, block=128):
    """x (R, K) -> q (R, K) float64 values, scales (Kb, R)."""
    x = np.asarray(x, np.float32)
    R, K = x.shape
    kb = -(-K // block)
    q, s = np.zeros((R, K)), np.zeros((kb, R))
    for r in range(R):
        for j in range(kb):
            sl = slice(j * block, min(K, (j + 1) * block))
            q[r, sl], s[j, r] = _round_block(x[r, sl])
    return q, s


def quantize_tiles(w, block=128):
    """w (N, K) -> q (N, K) float64 values, scales (Nb, Kb)."""
    w = np.asarray(w, np.float32)
    N, K = w.shape
    nb, kb = -(-N // block), -(-K // block)
    q, s = np.zeros((N, K)), np.zeros((nb, kb))
    for i in range(nb):
        for j in range(kb):
            sl = np.s_[i * block:min(N, (i + 1) * block), j * block:min(K, (j + 1) * block)]
            q[sl], s[i, j] = _round_block(w[sl])
    return q, s


def held_rows(q, s, block=128):
    """What rows in 8 bits stand for: q (R, K), s (Kb, R)."""
    return q * np.repeat(s.T, block, 1)[:, : q.shape[1]]


def held_tiles(q, s, block=128):
    return q * np.repeat(np.repeat(s, block, 0)[: q.shape[0]], block, 1)[:, : q.shape[1]]


def dropped(a, b, unit=2.0 ** -13, group=8):
    """What a product a (M, K) · b (N, K)ᵀ can lose where every `group`
    consecutive k are aligned to their largest product and cut at `unit` of
    it: of all but that one, less than unit · max each."""
    out = np.zeros((a.shape[0], b.shape[0]))
    for k in range(0, a.shape[1], group):
        m = np.zeros_like(out)
        for i in range(k, min(a.shape[1], k + group)):
            np.maximum(m, np.abs(a[:, i:i + 1]) * np.abs(b[:, i]), out=m)
        out += (group - 1) * unit * m
    return out


def experts(x, inds, gates, x_k, key, value, x_prev=None, residual=None, aligned=False):
    """The expert layer in 8 bits: key, value lists of what the weights stand
    for, (F, C) and (C, F).  The mixed and the hidden rows are fp32 values.
    Returns (out, Σ |gate| Σ |h| |v|, slack): slack bounds what `out` moves by
    where the products lose what `dropped` says (`aligned`).  A hidden value
    h = relu(z)² moves by at most 2 |z| d + d² with z's error d, and each of
    the two roundings to e4m3 is off by half a step, 2^-4 of the value or
    2^-10 of the block's factor."""
    x = np.asarray(x, np.float32)
    B, T, C = x.shape
    prev = np.zeros_like(x)
    prev[:, 1:] = x[:, :-1]
    if x_prev is not None:
        prev[:, 0] = np.asarray(x_prev, np.float32)
    out = np.zeros((B, T, C)) if residual is None else np.asarray(residual, np.float64).copy()
    size = np.zeros((B, T, C))
    slack = np.zeros((B, T, C))
    for b in range(B):
        for t in range(T):
            for j in range(inds.shape[2]):
                e = int(inds[b, t, j])
                if not 0 <= e < len(key):
                    continue
                m = x[b, t] + (prev[b, t] - x[b, t]) * np.asarray(x_k[e], np.float32)
                a = held_rows(*quantize_rows(m[None]))
                h = (a @ key[e].T)[0]
                z = np.abs(h)
                h = np.maximum(h.astype(np.float32), 0)
                hv = held_rows(*quantize_rows((h * h)[None]))[0]
                g = float(gates[b, t, j])
                out[b, t] += g * (hv @ value[e].T)
                size[b, t] += abs(g) * (np.abs(hv) @ np.abs(value[e]).T)
                if aligned:
                    kb = -(-C // 128)
                    d = dropped(a, key[e])[0] + 2.0 ** -23 * (128 + kb) * (np.abs(a) @ np.abs(key[e]).T)[0]
                    dh = 2 * z * d + d * d
                    top = np.repeat([(h * h + dh)[i:i + 128].max() for i in range(0, len(dh), 128)], 128)[:len(dh)]
                    dq = dh + (2 * h.astype(np.float64) ** 2 + dh) * 2.0 ** -4 + top / E4M3_MAX * 2.0 ** -9
                    v = np.abs(value[e])
                    # the value product loses its own share, of hidden rows that have moved by dq
                    slack[b, t] += abs(g) * (dq @ v.T + dropped(np.abs(hv)[None] + dq, v)[0]) * (1 + 2.0 ** -10)
    return out, size, slack
