"""Pages, rotary axes, norms, summaries and selections in 64 bits (whole numbers
where they are whole) on the CPU, from their definitions: the oracle of the tests
of drinkme_amd.kv_ops and norm_ops. Nothing here uses the package."""

from __future__ import annotations

import numpy as np

from tests import kv_reference as R

CAP = 2 ** 30 - 1


def reserve(free, count, table, lengths, new, page, total, pages):
    """On lists, in place; -> (cu, positions, slots, pages left, pages lacking)."""
    cu, positions, slots, lacking = [0], [-1] * total, [-1] * total, 0
    cols = len(table[0])
    for b, n in enumerate(new):
        n = min(max(n, 0), total - cu[-1])
        length = min(max(lengths[b], 0), CAP)
        for col in range(-(-length // page), min(cols, -(-(length + n) // page))):
            if count:
                count -= 1
                table[b][col] = free[count]
            else:
                table[b][col], lacking = -1, lacking + 1
        for m in range(n):
            p = length + m
            positions[cu[-1] + m] = p
            if p // page < cols and 0 <= table[b][p // page] < pages:
                slots[cu[-1] + m] = table[b][p // page] * page + p % page
        lengths[b] = length + n
        cu.append(cu[-1] + n)
    return cu, positions, slots, count, lacking


def trim(free, count, table, lengths, keep, page):
    """On lists, in place; -> pages left."""
    back = []
    for b, k in enumerate(keep):
        length = min(max(lengths[b], 0), CAP)
        k = min(max(k, 0), length)
        for col in range(-(-k // page), min(len(table[b]), -(-length // page))):
            if 0 <= table[b][col] < len(free):
                back.append(table[b][col])
            table[b][col] = -1
        lengths[b] = k
    for p in reversed(back):
        if count < len(free):
            free[count] = p
            count += 1
    return count


def rotate_axes(x, positions, axes, table, layout, dtype=np.float64):
    """x [T, H, D], positions [axes, T]: angle i of token t from table[positions[axes[i], t], i]."""
    n = len(axes)
    inside = (positions >= 0) & (positions < table.shape[0])
    cs = np.stack([np.where(inside[a][:, None], table[np.where(inside[a], positions[a], 0), i], np.nan)
                   for i, a in enumerate(axes)], 1).astype(dtype)
    x = np.asarray(x, dtype)
    out = x.copy()
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def standard(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdims=True)
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def summary(k):
    """k [tokens, D] -> (int [2, D], exponent byte): the bounds of a page's keys."""
    seen = ~np.isnan(k)
    some = seen.any(0)
    hi = np.where(some, np.where(seen, k, -np.inf).max(0, initial=-np.inf), 0.0)
    lo = np.where(some, np.where(seen, k, np.inf).min(0, initial=np.inf), 0.0)
    top = max(np.abs(hi).max(), np.abs(lo).max())
    e = -126
    while top > 127 * 2.0 ** e:
        e += 1
    return np.stack([np.ceil(hi / 2.0 ** e), np.floor(lo / 2.0 ** e)]).astype(np.int64), e + 127


def whole_queries(q):
    """q [group, D] -> whole numbers of one power of two, at most 127 of it."""
    q = np.where(np.isfinite(q), q, 0.0)
    top, e = np.abs(q).max(), -126
    while np.rint(top / 2.0 ** e) > 127:
        e += 1
    return np.rint(q / 2.0 ** e).astype(np.int64)


def score(q, bounds, scale):
    """The score of a page for queries [group, D], as fp32 has it."""
    w = whole_queries(q)
    s = (np.where(w > 0, w, 0) @ bounds[0] + np.where(w < 0, w, 0) @ bounds[1]).max()
    assert abs(s) < 2 ** 24
    with np.errstate(over="ignore"):
        return float(np.float32(np.ldexp(float(s), int(scale) - 127)))


def select(q, bounds, scales, pages, n, count, first, last):
    """q [group, D], bounds [pages, 2, D], scales [pages] of one head; `pages` of a
    sequence's columns (out of range: none) -> the columns, ascending, -1 behind."""
    keys = []
    for c in range(n):
        if c < first or c >= n - last:
            keys.append((0, 0.0, c))
        elif not 0 <= pages[c] < len(scales):
            keys.append((2, 0.0, c))
        else:
            keys.append((1, -score(q, bounds[pages[c]].astype(np.int64), scales[pages[c]]), c))
    best = sorted(c for *_, c in sorted(keys)[:count])
    return best + [-1] * (count - len(best))


def listed_attention(q, k, v, first, scale, blocks, page, causal=True):
    """As kv_reference.attention, over the positions of the listed columns: q [n, Hq,
    D], k and v [L, H, D], blocks [n, H, count]."""
    n, Hq, _ = q.shape
    L, H = k.shape[:2]
    parts = [np.zeros_like(q), np.full((n, Hq), -np.inf), np.zeros_like(q), np.zeros((n, Hq))]
    group = Hq // H
    for m in range(n):
        for h in range(H):
            at = np.flatnonzero(np.isin(np.arange(L) // page, blocks[m, h]))
            if causal:
                at = at[at <= first + m]
            heads = slice(h * group, (h + 1) * group)
            got = R.attention(q[m:m + 1, heads], k[at][:, h:h + 1], v[at][:, h:h + 1], 0, scale, causal=False)
            for part, one in zip(parts, got):
                part[m, heads] = one[0]
    return parts
