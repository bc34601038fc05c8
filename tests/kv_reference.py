"""The key/value cache's operators in 64 bits on the CPU, from their
definitions: the oracle of the tests of drinkme_amd.kv_ops. Nothing here uses
the package."""

from __future__ import annotations

import math

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
MIDS = (GRID[1:] + GRID[:-1]) / 2


def encode(x):
    """x [..., 32 n] -> (codes [..., 32 n], exponent bytes [..., n])."""
    y = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(y).all(-1)
    y = np.where(finite[..., None], y, 0.0)
    top = np.abs(y).max(-1)
    m, e = np.frexp(top)  # top = m 2^e, m in [1/2, 1): the smallest unit with top < 7 units
    unit = np.where(top > 0, e - 3 + (m >= 7 / 8), -125).clip(-125, 125)
    a = np.abs(y) / np.exp2(unit)[..., None]
    up, down = np.searchsorted(MIDS, a, side="right"), np.searchsorted(MIDS, a, side="left")
    code = np.where(up == down, up, up - up % 2)  # between two: the even one
    code = code + 8 * (y < 0)
    return code.reshape(x.shape).astype(np.uint8), np.where(finite, unit + 127, 255).astype(np.uint8)


def decode(code, e):
    """The values that codes [..., 32 n] and bytes [..., n] stand for."""
    v = GRID[code & 7] * np.where(code > 7, -1.0, 1.0)
    scale = np.where(e == 255, np.nan, np.exp2(e.astype(np.float64) - 127))
    return (v.reshape(*code.shape[:-1], -1, 32) * scale[..., None]).reshape(code.shape)


def cached(x):
    return decode(*encode(x))


def rotate(x, positions, table, layout, dtype=np.float64):
    """x [T, H, D] by table [positions, angles, 2]; in float32 each product and
    sum is rounded, as the operator defines."""
    x, half = np.asarray(x, dtype), table.shape[1]
    out = x.copy()
    cs = np.asarray(table, dtype)[positions]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def attention(q, k, v, first, scale, causal=True, window=None):
    """q [n, Hq, D], its row m at position first + m, over k, v [L, H, D] ->
    (out, lse, weights' sum of |v|, largest sum of |q k| a row): float64. What a
    row does not see does not reach it."""
    n, Hq, D = q.shape
    L, H = k.shape[:2]
    out, lse = np.zeros((n, Hq, D)), np.full((n, Hq), -np.inf)
    spread, reach = np.zeros((n, Hq, D)), np.zeros((n, Hq))
    for m in range(n):
        hi = min(L, first + m + 1) if causal else L
        lo = max(0, first + m + 1 - window) if window else 0
        if hi <= lo:
            continue
        for g in range(Hq):
            kk, vv = k[lo:hi, g // (Hq // H)], v[lo:hi, g // (Hq // H)]
            s = scale * (kk @ q[m, g])
            if np.isnan(s).any():
                out[m, g], lse[m, g] = np.nan, np.nan
                continue
            top = s.max()
            w = np.exp(s - top)
            lse[m, g] = top + math.log(w.sum())
            w /= w.sum()
            out[m, g], spread[m, g] = w @ vv, w @ np.abs(vv)
            reach[m, g] = scale * (np.abs(kk) @ np.abs(q[m, g])).max()
    return out, lse, spread, reach


def bound(out, spread, reach, tokens, dim, bf16):
    """How far a result may be from attention()'s `out`: scores summed in fp32
    (dim products each 2^-24 off, twice: in the numerator and the sum), weights
    by exp2 and sums of up to `tokens` terms in fp32, the weights rounded to
    bf16 (2^-8 of each) or carried in 24 bits, and the result's own rounding."""
    scores = 2 * (dim + 4) * 2.0 ** -24 * reach[..., None]
    sums = (tokens + 64) * 2.0 ** -24
    weights, last = (2.0 ** -8, 2.0 ** -8) if bf16 else (2.0 ** -23, 2.0 ** -24)
    return (scores + sums + weights) * spread * 1.01 + last * np.abs(out) * 1.01 + 1e-37


def lse_bound(lse, reach, tokens, dim):
    return 2 * (dim + 4) * 2.0 ** -24 * reach + (tokens + 64) * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(np.isfinite(lse), lse, 0)) + 1e-6
