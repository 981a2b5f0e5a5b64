"""Float64 definitions of the training operators, straight from their formulas:
attention with a learned relative position bias and its gradients, the bias by itself,
the orthogonalised update.  NumPy loops over heads; nothing of the package is used."""

from __future__ import annotations

import numpy as np


def line_row(rel: int, num_buckets: int, max_distance: int, bidirectional: bool) -> int:
    """Row of the pair whose key is ``rel`` positions after its query."""
    n, base = num_buckets, 0
    if bidirectional:
        n //= 2
        if rel > 0:
            base = n
        dist = abs(rel)
    else:
        dist = max(0, -rel)
    half = n // 2
    if dist < half:
        return base + dist
    # the last j with dist >= half * (max_distance / half) ** (j / (n - half)), raised
    # to the power n - half so that both sides are whole numbers
    wide, j = n - half, 0
    while j + 1 < wide and dist ** wide >= half ** (wide - j - 1) * max_distance ** (j + 1):
        j += 1
    return base + half + j


def line_rows(q_len, k_len, q_start=0, num_buckets=32, max_distance=128, bidirectional=True):
    lo, hi = -(q_start + q_len - 1), k_len - 1 - q_start
    by_rel = np.array([line_row(r, num_buckets, max_distance, bidirectional)
                       for r in range(lo, hi + 1)])
    return by_rel[np.arange(k_len)[None] - (q_start + np.arange(q_len))[:, None] - lo]


def grid_rows(height, width):
    t = np.arange(height * width)
    dy = (t // width)[:, None] - (t // width)[None]
    dx = (t % width)[:, None] - (t % width)[None]
    return (dy + height - 1) * (2 * width - 1) + dx + width - 1


def visible(batch, heads, q_len, k_len, *, causal=False, mask=None, key_lengths=None, q_start=0):
    """(batch, heads, q_len, k_len) booleans."""
    see = np.ones((batch, heads, q_len, k_len), dtype=bool)
    j = np.arange(k_len)
    start = np.broadcast_to(np.asarray(q_start), (batch,))
    if causal:
        see &= (j <= (start[:, None] + np.arange(q_len))[..., None])[:, None]
    if key_lengths is not None:
        see &= (j < np.asarray(key_lengths)[:, None])[:, None, None]
    if mask is not None:
        m = np.asarray(mask)
        m = m[None, None] if m.ndim == 2 else m
        see &= m[np.arange(batch) % m.shape[0]]
    return see


def attention(q, k, v, table, rows, see, scale, dout=None):
    """out, and with ``dout`` also dq, dk, dv, dtable.  ``rows``: (q_len, k_len), or one
    such array for each batch entry.  Places that nothing sees may hold anything."""
    q, k, v, table = (np.asarray(t, dtype=np.float64) for t in (q, k, v, table))
    b, h, lq, d = q.shape
    group = h // k.shape[1]
    out = np.zeros(q.shape)
    grads = [np.zeros(t.shape) for t in (q, k, v, table)]
    for n in range(b):
        rw = rows if rows.ndim == 2 else rows[n]
        for m in range(h):
            s_ = see[n, m]
            qq = np.where(s_.any(1)[:, None], q[n, m], 0.0)
            kk = np.where(s_.any(0)[:, None], k[n, m // group], 0.0)
            vv = np.where(s_.any(0)[:, None], v[n, m // group], 0.0)
            s = np.where(s_, scale * (qq @ kk.T) + table[:, m][rw], -np.inf)
            top = s.max(1, keepdims=True)
            p = np.exp(s - np.where(np.isinf(top), 0.0, top))
            total = p.sum(1, keepdims=True)
            p = p / np.where(total == 0, 1.0, total)
            out[n, m] = p @ vv
            if dout is None:
                continue
            g = np.where(s_.any(1)[:, None], np.asarray(dout, dtype=np.float64)[n, m], 0.0)
            dp = g @ vv.T
            ds = p * (dp - (p * dp).sum(1, keepdims=True))
            grads[0][n, m] = scale * ds @ kk
            grads[1][n, m // group] += scale * ds.T @ qq
            grads[2][n, m // group] += p.T @ g
            np.add.at(grads[3][:, m], rw, ds)
    return out if dout is None else (out, *grads)


def bias(table, rows):
    return np.moveaxis(np.asarray(table, dtype=np.float64)[rows], -1, 0)


def bias_grad(up, rows, table_rows):
    up = np.asarray(up, dtype=np.float64)
    out = np.zeros((table_rows, up.shape[0]))
    for m in range(up.shape[0]):
        np.add.at(out[:, m], rows, up[m])
    return out


def orthogonalize(g, steps, coefficients, eps=1e-7):
    a, b, c = coefficients
    x = np.asarray(g, dtype=np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.sqrt((x * x).sum()) + eps)
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.T if tall else x
