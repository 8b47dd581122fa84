"""64-bit restatements of the operators around the expert block: norm, 8-bit
product, rotary positions into a paged cache, paged attention.

TEST INFRASTRUCTURE ONLY.  Plain numpy on float64 arrays, written from the
operators' definitions; nothing is rounded except where the definition names a
stored type.  The reference has no counterpart of these operators (its engines
take them from their model library): parity unpinned, the definitions are the
oracle.
"""
from __future__ import annotations

import numpy as np

FP8_MAX = 448.0
FP8_LEAST = 1e-30


def e4m3(v) -> np.ndarray:
    """Values in [-448, 448] (a little over counts as 448) -> nearest e4m3, ties to even."""
    v = np.asarray(v, dtype=np.float64)
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6)))
    step = np.exp2(np.minimum(e, 8.0) - 3)
    return np.rint(v / step) * step


def quant(y):
    """[T, D] -> (codes' values, scales [T, ceil(D / 128)])."""
    T, D = y.shape
    nb = -(-D // 128)
    q, s = np.empty((T, D)), np.empty((T, nb))
    for b in range(nb):
        c = slice(128 * b, min(D, 128 * b + 128))
        most = np.maximum(np.abs(y[:, c]).max(1), FP8_LEAST)
        s[:, b] = most / FP8_MAX
        q[:, c] = e4m3(y[:, c] * FP8_MAX / most[:, None])
    return q, s


def rms_norm(h, w, eps):
    return h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w


def linear(xq, xs, wq, ws):
    """(y, sum of the products' magnitudes), both [T, N]."""
    K, N = xq.shape[1], wq.shape[0]
    col = np.arange(K) // 128
    a = xq * xs[:, col]
    b = wq * ws[np.arange(N) // 128][:, col]
    return a @ b.T, np.abs(a) @ np.abs(b).T


def turn(x, pos, freqs, mscale, interleaved):
    """x [n, heads, D] at positions pos [n] -> rotated."""
    y = x.copy()
    R = len(freqs)
    ang = pos[:, None].astype(np.float64) * freqs
    c, s = mscale * np.cos(ang)[:, None], mscale * np.sin(ang)[:, None]
    i = np.arange(R)
    i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + R)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def attention(q, k, v, pos, scale, window, sinks):
    """q [n, H, D] at positions pos; k, v [L, HK, D] -> (out, the sum of p |v| / sum of
    p): rows that see nothing are zero."""
    n, H, D = q.shape
    L, HK, _ = k.shape
    out, mag = np.zeros((n, H, D)), np.zeros((n, H, D))
    j = np.arange(L)
    for i in range(n):
        seen = j <= pos[i]
        if window:
            seen &= j > pos[i] - window
        if not seen.any():
            continue
        ks, vs = k[seen], v[seen]
        for h in range(H):
            g = h // (H // HK)
            z = ks[:, g] @ q[i, h] * scale
            m = max(z.max(), sinks[h]) if sinks is not None else z.max()
            p = np.exp(z - m)
            d = p.sum() + (np.exp(sinks[h] - m) if sinks is not None else 0.0)
            out[i, h] = p @ vs[:, g] / d
            mag[i, h] = p @ np.abs(vs[:, g]) / d
    return out, mag
