"""Plain float64 restatements of the token operators (layer norm, rotary
positions, attention over packed sequences) and of their gradients, one row,
head and sequence at a time, from the definitions alone. CPU, numpy."""

from __future__ import annotations

import numpy as np


# -------------------------------------------------------------------- norm

def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """y of rows x (rows, n)."""
    x = np.asarray(x, np.float64)
    m = x.mean(1, keepdims=True)
    y = (x - m) / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + eps)
    y = y if weight is None else y * weight
    return y if bias is None else y + bias


def layer_norm_grad(x, weight, dy, eps=1e-5):
    """(dx, dweight, dbias), each row by its Jacobian."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    n = x.shape[1]
    w = np.ones(n) if weight is None else np.asarray(weight, np.float64)
    dx, dw = np.zeros_like(x), np.zeros(n)
    for r in range(x.shape[0]):
        c = x[r] - x[r].mean()
        s = 1.0 / np.sqrt((c ** 2).mean() + eps)
        u = c * s
        g = dy[r] * w
        dx[r] = s * (g - g.mean() - u * (g * u).mean())
        dw += dy[r] * u
    return dx, dw, dy.sum(0)


# ------------------------------------------------------------------ rotary

def rotary(x, positions, frequencies, layout, inverse=False):
    """x (tokens, heads, dim) turned; positions (tokens, axes)."""
    y = np.array(x, np.float64)
    pairs, axes = len(frequencies), positions.shape[1]
    for i in range(pairs):
        a, b = (i, pairs + i) if layout == "half" else (2 * i, 2 * i + 1)
        t = positions[:, i // (pairs // axes)].astype(np.float64) * frequencies[i]
        c, s = np.cos(t)[:, None], np.sin(t)[:, None] * (-1.0 if inverse else 1.0)
        p, q = np.array(x[..., a], np.float64), np.array(x[..., b], np.float64)
        y[..., a], y[..., b] = p * c - q * s, q * c + p * s
    return y


# --------------------------------------------------------------- attention

def sees(nq, nk, causal):
    """(nq, nk) truth values: query i stands at key i + nk - nq."""
    if not causal:
        return np.ones((nq, nk), bool)
    return np.arange(nk)[None, :] <= np.arange(nq)[:, None] + (nk - nq)


def probabilities(q, k, scale, mask):
    """Softmax over the seen keys of one head; rows that see none are zeros."""
    s = np.where(mask, scale * (q @ np.where(np.isfinite(k), k, 0.0).T), -np.inf)
    top = s.max(1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = p.sum(1, keepdims=True)
    return p / np.where(total == 0.0, 1.0, total)


def attention(q, k, v, q_offsets, k_offsets, causal, scale, dout=None, unit=0.0):
    """(o, dq, dk, dv) and, as a second tuple, how far each may be off when o and
    the gradients are rounded to a type of unit roundoff `unit` and p and ds are
    rounded to it for their products, sums being exact: first order, every
    rounding at its worst and alike in sign.

    o: unit (|o| + p |v|). delta = do o takes o's error: e_i = |do_i| (that).
    dv: unit (|dv| + p^T |do|). dq: unit (|dq| + scale |ds| |k|) + scale e p |k|,
    and dk the same with q."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out = [np.zeros(t.shape) for t in (q, q, k, v)]
    off = [np.zeros(t.shape) for t in (q, q, k, v)]
    for q0, q1, k0, k1 in zip(q_offsets[:-1], q_offsets[1:], k_offsets[:-1], k_offsets[1:]):
        rows, keys = slice(q0, q1), slice(k0, k1)
        mask = sees(q1 - q0, k1 - k0, causal)
        for h in range(q.shape[1]):
            qh, kh, vh = q[rows, h], k[keys, h // group], v[keys, h // group]
            p = probabilities(qh, kh, scale, mask)
            kf, vf = np.where(np.isfinite(kh), kh, 0.0), np.where(np.isfinite(vh), vh, 0.0)
            o = p @ vf
            out[0][rows, h] = o
            o_off = unit * (np.abs(o) + p @ np.abs(vf))
            off[0][rows, h] = o_off
            if dout is None:
                continue
            do = np.asarray(dout, np.float64)[rows, h]
            delta = (do * o).sum(1, keepdims=True)
            ds = p * (do @ vf.T - delta)
            e = (np.abs(do) * o_off).sum(1, keepdims=True)
            out[1][rows, h] = scale * ds @ kf
            off[1][rows, h] = scale * (unit * np.abs(ds) @ np.abs(kf) + e * (p @ np.abs(kf)))
            out[2][keys, h // group] += scale * ds.T @ qh
            off[2][keys, h // group] += scale * (unit * np.abs(ds).T @ np.abs(qh) +
                                                 (e * p).T @ np.abs(qh))
            out[3][keys, h // group] += p.T @ do
            off[3][keys, h // group] += unit * p.T @ np.abs(do)
    for i in (1, 2, 3):
        off[i] += unit * np.abs(out[i])
    return tuple(out), tuple(off)
