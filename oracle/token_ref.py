"""Plain float64 restatements of the token operators (layer norm, rotary
positions, heads normed and turned, dropout, attention over packed sequences) and
of their gradients, one row, head and sequence at a time, from the definitions
alone. CPU, numpy."""

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


def axes_of(sections, order):
    """The axis of each pair: each axis's pairs as neighbours ("runs"), or pair after
    pair dealt to the axes that have pairs left ("turns")."""
    if order == "runs":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [a for n in range(max(sections)) for a in range(len(sections)) if n < sections[a]]


def rotary_axes(x, positions, frequencies, layout, axes, inverse=False):
    """`rotary` with pair i going by positions[:, axes[i]]."""
    return rotary(x, np.asarray(positions)[:, axes], frequencies, layout, inverse)


# ------------------------------------------------------- heads normed and turned

def norm_rotary(x, weight, eps, turn):
    """turn(x / sqrt(mean(x^2) + eps) * weight), of heads x (tokens, heads, dim)."""
    x = np.asarray(x, np.float64)
    u = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    return turn(u if weight is None else u * weight)


def norm_rotary_grad(x, weight, eps, turn_back, dy):
    """(dx, dweight), each head by its Jacobian."""
    x, n = np.asarray(x, np.float64), x.shape[-1]
    w = np.ones(n) if weight is None else np.asarray(weight, np.float64)
    g = turn_back(np.asarray(dy, np.float64))
    dx, dw = np.zeros_like(x), np.zeros(n)
    for t in range(x.shape[0]):
        for h in range(x.shape[1]):
            s = 1.0 / np.sqrt((x[t, h] ** 2).mean() + eps)
            u = x[t, h] * s
            d = g[t, h] * w
            dx[t, h] = s * (d - u * (d * u).mean())
            dw += g[t, h] * u
    return dx, dw


# ----------------------------------------------------------------- dropout

def philox4x32(counter, key):
    """One block of Philox4x32-10: four words of 32 bits of four and two."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(n, drop, seed, site=0, first=0):
    """Truth values of elements first .. first + n - 1: 16 bits of the block of every
    eight, at least `drop`."""
    out = []
    for i in range(first, first + n):
        w = philox4x32((i // 8 & 0xFFFFFFFF, i // 8 >> 32, site & 0xFFFFFFFF, site >> 32),
                       (seed & 0xFFFFFFFF, seed >> 32))[i % 8 // 2]
        out.append((w >> 16 if i % 2 else w & 0xFFFF) >= drop)
    return np.array(out, bool)


# --------------------------------------------------------------- attention

def sees(nq, nk, causal, window=None, sinks=0):
    """(nq, nk) truth values: query i stands at key i + nk - nq; with a window it sees
    the last `window` keys up to there and the first `sinks`."""
    if not causal:
        return np.ones((nq, nk), bool)
    key, at = np.arange(nk)[None, :], np.arange(nq)[:, None] + (nk - nq)
    seen = key <= at
    return seen if window is None else seen & ((key > at - window) | (key < sinks))


def probabilities(q, k, scale, mask):
    """Softmax over the seen keys of one head; rows that see none are zeros."""
    s = np.where(mask, scale * (q @ np.where(np.isfinite(k), k, 0.0).T), -np.inf)
    top = s.max(1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = p.sum(1, keepdims=True)
    return p / np.where(total == 0.0, 1.0, total)


def attention(q, k, v, q_offsets, k_offsets, causal, scale, dout=None, unit=0.0, window=None,
              sinks=0):
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
        mask = sees(q1 - q0, k1 - k0, causal, window, sinks)
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


def shared_attention(q, k, v, shared_k, shared_v, q_offsets, k_offsets, group_offsets,
                     shared_offsets, causal, scale, unit=0.0):
    """o and how far it may be off (as `attention`): each query over its group's shared
    keys and the keys that it sees of its own sequence."""
    q, k, v, sk, sv = (np.asarray(t, np.float64) for t in (q, k, v, shared_k, shared_v))
    group = q.shape[1] // k.shape[1]
    out, off = np.zeros(q.shape), np.zeros(q.shape)

    def bounds(offsets, token):
        """The sequence that has a token, or -1."""
        for s in range(len(offsets) - 1):
            if offsets[s] <= token < offsets[s + 1]:
                return s
        return -1

    for t in range(q.shape[0]):
        s, g = bounds(q_offsets, t), bounds(group_offsets, t)
        own = np.arange(0)
        if s >= 0:
            own = np.arange(k_offsets[s], k_offsets[s + 1])
            if causal:
                own = own[:max(0, t - q_offsets[s + 1] + 1 + len(own))]
        all_shared = np.arange(0) if g < 0 else np.arange(shared_offsets[g], shared_offsets[g + 1])
        if len(own) + len(all_shared) == 0:
            continue
        for h in range(q.shape[1]):
            kh = np.concatenate([sk[all_shared, h // group], k[own, h // group]])
            vh = np.concatenate([sv[all_shared, h // group], v[own, h // group]])
            p = probabilities(q[t:t + 1, h], kh, scale, np.ones((1, len(kh)), bool))[0]
            out[t, h] = p @ vh
            off[t, h] = unit * (np.abs(out[t, h]) + p @ np.abs(vh))
    return out, off
