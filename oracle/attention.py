"""Sliding-window attention with sinks in 64 bits, with the error a float32-accumulating kernel may have.

``forward`` and ``backward`` take NumPy arrays [batch, heads, tokens, head_dim] and follow the
definition: key j is visible to the query at position p = offset + i when j < length, j <= p and
(no window, or p - j < window, or j < sinks); a row without visible keys gives zeros.

``tolerances`` bounds |kernel - oracle| elementwise from the arithmetic alone. With u = 2^-24
(float32) and t the unit roundoff of the stored type (the weights P and dS are rounded to it for
the products, t = u for float32):

* a score is a float32 sum of D products: eps_s = (D + 4) u max(scale sum |q||k|); a weight then
  has the relative error eps_p = 2 eps_s + 16 u (the score's and the normaliser's, the
  exponential's and the sums' roundings);
* o = sum P v with sum P = 1: (eps_p + t + n u) max|v| + t |o|;
* dP: eps_dp = (D + 4) u max(sum |g||v|); delta uses the stored o:
  eps_delta = (D u + o's relative error) max(sum |g||o|) + max|g|_1 times o's absolute error;
* dS = P (dP - delta): per unit of P, eps_ds = (eps_p + t) max|dP - delta| + eps_dp + eps_delta;
* dq: scale max|k| (eps_ds + n u max|dP - delta|) + t |dq| (rows of P sum to 1); dk and dv: the same
  per unit of column sum of P over the queries and the heads of the group.

* float16 numbers below the normal range lose up to 2^-25 each. The forward's weights: n times that, times
  the largest factor, per output. The backward's weights are held times 2^14, and dS times a power of two
  that brings 2 max|g|_2 max|v|_2 to 2^13 at least: n 2^-39 and n 2^-37 of that product.

Everything is doubled for the terms of second order.
"""
from __future__ import annotations

import numpy as np

UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# Half the spacing of float16's subnormal numbers (nothing comparable in the other types).
FLOOR = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}


def visible(queries, keys, length, window, sinks, offset=0):
    """[queries, keys] bool."""
    p, j = offset + np.arange(queries)[:, None], np.arange(keys)[None, :]
    seen = (j < length) & (j <= p)
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


def _weights(q, k, seen, scale):
    s = scale * (q @ k.T)
    s = np.where(seen, s, -np.inf)
    top = s.max(axis=1, initial=-np.inf, keepdims=True)
    e = np.exp(s - np.where(np.isinf(top), 0.0, top))
    total = e.sum(axis=1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    with np.errstate(divide="ignore"):
        lse = np.where(total[:, 0] == 0, -np.inf, np.where(np.isinf(top[:, 0]), 0.0, top[:, 0]) + np.log(total[:, 0]))
    return p, lse


def _clean(x, length):
    """float64 with zeros at and past the length (whatever is there has no effect)."""
    x = np.array(x, np.float64)
    x[length:] = 0.0
    return x


def forward(q, k, v, *, window=0, sinks=0, lengths=None, offset=0, scale=None):
    """(output, lse)."""
    batch, heads, queries, dim = q.shape
    group, keys = heads // k.shape[1], k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, lse = np.zeros(q.shape, np.float64), np.zeros((batch, heads, queries))
    for b in range(batch):
        length = keys if lengths is None else int(np.clip(lengths[b], 0, keys))
        seen = visible(queries, keys, length, window, sinks, offset)
        for h in range(heads):
            p, lse[b, h] = _weights(q[b, h].astype(np.float64), _clean(k[b, h // group], length), seen, scale)
            out[b, h] = p @ _clean(v[b, h // group], length)
    return out, lse


def backward(q, k, v, g, *, window=0, sinks=0, lengths=None, offset=0, scale=None):
    """(dq, dk, dv)."""
    batch, heads, queries, dim = q.shape
    group, keys = heads // k.shape[1], k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for b in range(batch):
        length = keys if lengths is None else int(np.clip(lengths[b], 0, keys))
        seen = visible(queries, keys, length, window, sinks, offset)
        for h in range(heads):
            m = h // group
            qq, gg = q[b, h].astype(np.float64), g[b, h].astype(np.float64)
            kk, vv = _clean(k[b, m], length), _clean(v[b, m], length)
            p, _ = _weights(qq, kk, seen, scale)
            dp = gg @ vv.T
            ds = p * (dp - (p * dp).sum(axis=1, keepdims=True)) * scale
            dq[b, h] = ds @ kk
            dk[b, m] += ds.T @ qq
            dv[b, m] += p.T @ gg
    return dq, dk, dv


def tolerances(q, k, v, dtype, g=None, *, window=0, sinks=0, lengths=None, offset=0, scale=None):
    """Bounds for (out, lse) or, with g, for (out, lse, dq, dk, dv), each of its array's shape."""
    batch, heads, queries, dim = q.shape
    group, keys = heads // k.shape[1], k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    u, t, floor = 2.0 ** -24, UNIT[dtype], FLOOR[dtype]
    n = max(keys, queries * group)
    k64 = np.stack([np.stack([_clean(x, keys if lengths is None else int(np.clip(lengths[b], 0, keys))) for x in k[b]])
                    for b in range(batch)]) if batch else np.zeros(k.shape)
    v64 = np.stack([np.stack([_clean(x, keys if lengths is None else int(np.clip(lengths[b], 0, keys))) for x in v[b]])
                    for b in range(batch)]) if batch else np.zeros(v.shape)
    q64 = q.astype(np.float64)
    rep = lambda x: np.repeat(x, group, axis=1)  # noqa: E731
    top = lambda x: float(np.max(x, initial=0.0))  # noqa: E731
    out, lse = forward(q, k, v, window=window, sinks=sinks, lengths=lengths, offset=offset, scale=scale)
    scores = top(scale * np.abs(q64) @ np.abs(rep(k64)).swapaxes(-1, -2))
    eps_s = (dim + 4) * u * scores
    eps_p = 2 * eps_s + 16 * u
    out_abs = (eps_p + t + n * u + n * floor) * top(np.abs(v64))
    t_out = 2 * (out_abs + t * np.abs(out)) + floor
    t_lse = np.full(lse.shape, 2 * (eps_s + 16 * u + 4 * u * (scores + 16)))
    if g is None:
        return t_out, t_lse
    g64 = g.astype(np.float64)
    dq, dk, dv = backward(q, k, v, g, window=window, sinks=sinks, lengths=lengths, offset=offset, scale=scale)
    dp = top(np.abs(g64) @ np.abs(rep(v64)).swapaxes(-1, -2))
    eps_dp = (dim + 4) * u * dp
    g_sum = top(np.abs(g64).sum(-1))
    eps_delta = dim * u * top((np.abs(g64) * np.abs(out)).sum(-1)) + g_sum * (out_abs + t * top(np.abs(out)))
    spread = 2 * dp
    eps_ds = (eps_p + t) * spread + eps_dp + eps_delta
    columns = np.zeros((batch, k.shape[1], keys, 1))
    for b in range(batch):
        length = keys if lengths is None else int(np.clip(lengths[b], 0, keys))
        seen = visible(queries, keys, length, window, sinks, offset)
        for h in range(heads):
            p, _ = _weights(q64[b, h], k64[b, h // group], seen, scale)
            columns[b, h // group, :, 0] += p.sum(axis=0)
    per = eps_ds + n * u * spread
    norm = lambda x: top(np.linalg.norm(x, axis=-1))  # noqa: E731
    lost = n * floor * 2.0 ** -12 * 2 * norm(g64) * norm(v64)
    t_dq = 2 * (scale * top(np.abs(k64)) * (per + lost) + t * np.abs(dq)) + floor
    t_dk = 2 * (scale * top(np.abs(q64)) * (per * columns + lost) + t * np.abs(dk)) + floor
    t_dv = 2 * (((eps_p + t + n * u) * columns + n * floor * 2.0 ** -14) * top(np.abs(g64)) + t * np.abs(dv)) + floor
    return t_out, t_lse, t_dq, t_dk, t_dv
