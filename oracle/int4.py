"""64-bit oracle of the 4-bit cache, attention over it and the 4-bit-weight linear (numpy).

16-bit scales and activations arrive as float64 arrays of their exact values; ``mant`` is the number
of mantissa bits of the 16-bit type (7 for bf16, 10 for fp16), ``emin`` its least normal exponent."""
from __future__ import annotations

import numpy as np

D = 128
MANT = {"bf16": (7, -126), "fp16": (10, -14)}


def round16(x, kind):
    """Nearest value of the 16-bit type (ties to even), as float64; no overflow handling."""
    mant, emin = MANT[kind]
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 1, emin).astype(np.float64) - mant)
    return np.rint(x / step) * step


def key_dim(place):
    """Dim of the key at half byte ``place`` (0 .. 127) of its 64 bytes."""
    word, p = divmod(place, 8)
    g, i = divmod(word, 4)
    return 32 * i + 8 * g + 2 * (p % 4) + p // 4


def value_dim(place):
    word, t = divmod(place, 8)
    return 16 * t + word


def unpack(row, dim_of):
    """(..., 64) bytes -> (..., 128) codes by dim."""
    out = np.empty((*row.shape[:-1], D), dtype=np.int64)
    for place in range(D):
        b = row[..., place // 2].astype(np.int64)
        out[..., dim_of(place)] = (b >> 4 if place & 1 else b) & 15
    return out


def values(codes, scales):
    """Cached rows (..., 128 bytes), (..., 4 NG) -> (key, value) (..., 128) in 64 bits."""
    ng = scales.shape[-1] // 4
    out = []
    for part, dim_of in ((0, key_dim), (1, value_dim)):
        c = unpack(codes[..., 64 * part:64 * part + 64], dim_of)
        sz = scales[..., 2 * ng * part:2 * ng * (part + 1)]
        s = np.repeat(sz[..., 0::2], D // ng, -1)
        z = np.repeat(sz[..., 1::2], D // ng, -1)
        out.append(z + s * c)
    return out


def norm_rotate(x, w, eps, cos, sin):
    """x (T, H, 128), cos / sin (T, 64): RMSNorm with w (None: none), then rotate-half."""
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w
    a, b = x[..., :64], x[..., 64:]
    c, s = cos[:, None, :], sin[:, None, :]
    return np.concatenate((a * c - b * s, b * c + a * s), -1)


def attention(q, key, value, scale, first=None):
    """q (R, 128), key / value (L, 128); row r sees keys [0, first + r] (None: all). Returns the
    output, and sum_j p_j |v_j|-like weights p (R, L)."""
    s = (q @ key.T) * scale
    if first is not None:
        seen = np.arange(key.shape[0])[None, :] <= first + np.arange(q.shape[0])[:, None]
        s = np.where(seen, s, -np.inf)
    m = s.max(-1, keepdims=True) if s.shape[1] else np.zeros((s.shape[0], 1))
    p = np.exp(s - np.where(np.isfinite(m), m, 0))
    l = p.sum(-1, keepdims=True)
    p = np.divide(p, l, out=np.zeros_like(p), where=l > 0)
    return p @ value, p


def weights(qweight, scale):
    """(N, K / 2) bytes and (N, K / group) scales -> (N, K) in 64 bits."""
    n, half = qweight.shape
    w = np.empty((n, 2 * half))
    w[:, 0::2] = (qweight & 15).astype(np.float64) - 8
    w[:, 1::2] = (qweight >> 4).astype(np.float64) - 8
    return w * np.repeat(scale, 2 * half // scale.shape[1], -1)
