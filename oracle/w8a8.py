"""Oracle of the 8-bit activations and the integer linears (numpy).

16-bit inputs arrive as float32 arrays of their exact values. The codes follow from fp32 v and max |v| by one quotient
rounded to fp32. Of two 16-bit values, a 2^i and b 2^j with whole a and b below 2^11, the quotient 127 a / (b 2^f) is a
tie (2 n + 1) / 2 or differs from it by at least 1 / (b 2^(f + 1)), that is by 1 / (254 a) > 2^-19 of itself; fp32 moves
it by 2^-24 at most, so that this rounding moves no code. So they are compared for equality; scales and outputs in 64
bits, the linear's also by its own fp32 steps."""
from __future__ import annotations

import numpy as np


def codes(v):
    """v (rows, K) float32 -> (int64 codes, max |v| float64 (rows,)); rows with a NaN or an infinity: codes 0, NaN."""
    v = np.asarray(v, dtype=np.float32).astype(np.float64)
    most = np.abs(v).max(-1)
    fine = np.isfinite(most)
    safe = np.where(fine & (most > 0), most, 1.0)
    c = np.rint((127 * np.where(fine[:, None], v, 0) / safe[:, None]).astype(np.float32)).astype(np.int64)
    return np.where((fine & (most > 0))[:, None], c, 0), np.where(fine, most, np.nan)


def norm_products(x, w, residual=None):
    """s = x (+ residual) and s w, each rounded to fp32 as the operator does."""
    with np.errstate(over="ignore", invalid="ignore"):
        s = x.astype(np.float32) if residual is None else x.astype(np.float32) + residual.astype(np.float32)
        return s, s * w.astype(np.float32)


def norm_scale(most, s, eps):
    """max |v| / 127 times 1 / sqrt(mean(s^2) + eps), 64 bits."""
    s = s.astype(np.float64)
    return most / 127 / np.sqrt((s * s).mean(-1) + eps)


def _sums(x, w):
    """Whole numbers below 2^53, so that 64-bit floats hold every partial sum."""
    return x.astype(np.float64) @ w.astype(np.float64).T


def linear32(x, x_scale, w, scale, bias=None):
    """The operator's own arithmetic: exact integer sums, times scale in fp32, then times x_scale plus bias with one
    rounding to fp32 (through 64 bits of mantissa). float32, not rounded to the output's type."""
    y = _sums(x, w).astype(np.float32) * scale.astype(np.float32)[None]
    y = y.astype(np.longdouble) * x_scale.astype(np.longdouble)[:, None]
    return (y if bias is None else y + bias.astype(np.longdouble)[None]).astype(np.float32)


def linear64(x, x_scale, w, scale, bias=None):
    y = _sums(x, w) * scale.astype(np.float64)[None] * x_scale.astype(np.float64)[:, None]
    return y if bias is None else y + bias.astype(np.float64)[None]


def silu_up(y):
    """silu(gate) * up of y = [gate | up] (64 bits)."""
    gate, up = np.split(y, 2, axis=-1)
    return gate / (1 + np.exp(-gate)) * up
