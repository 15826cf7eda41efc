"""Counter-based dropout in NumPy: the Philox4x32 generator (Salmon, Moraes, Dror, Shaw 2011) and
residual + keep (x + bias) / (1 - p) with its gradients, in 64 bits."""
from __future__ import annotations

import numpy as np

_LOW = np.uint64(0xFFFFFFFF)
_SHIFT = np.uint64(32)


def philox4x32(counter, key, rounds):
    """counter: uint64 [n, 4] of 32-bit words, key: two 32-bit ints -> uint64 [n, 4]."""
    a, b, c, d = (np.asarray(counter, np.uint64)[:, i] for i in range(4))
    k0, k1 = (int(k) for k in key)
    for _ in range(rounds):
        x, y = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (y >> _SHIFT) ^ b ^ np.uint64(k0), y & _LOW, (x >> _SHIFT) ^ d ^ np.uint64(k1), x & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([a, b, c, d], axis=1)


def keep_mask(shape, p, seed, offset):
    """Bool array: True where the element is kept."""
    n = int(np.prod(shape))
    group = np.arange((n + 3) // 4, dtype=np.uint64)
    counter = np.stack([group & _LOW, group >> _SHIFT, np.full_like(group, offset & 0xFFFFFFFF),
                        np.full_like(group, offset >> 32)], axis=1)
    words = philox4x32(counter, (seed & 0xFFFFFFFF, seed >> 32), 7).reshape(-1)[:n]
    return (words >= np.uint64(int(p * 2.0 ** 32))).reshape(shape)


def forward(x, p, seed, offset, bias=None, residual=None):
    x = np.asarray(x, np.float64)
    if bias is not None:
        x = x + np.asarray(bias, np.float64)
    y = np.where(keep_mask(x.shape, p, seed, offset), x / (1.0 - p), 0.0)
    return y if residual is None else y + np.asarray(residual, np.float64)


def backward(g, p, seed, offset):
    """(dx, dbias)."""
    g = np.asarray(g, np.float64)
    dx = np.where(keep_mask(g.shape, p, seed, offset), g / (1.0 - p), 0.0)
    return dx, dx.reshape(-1, g.shape[-1]).sum(axis=0)
