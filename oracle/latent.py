"""Laws of rotary positions, the latent cache and its attention on the host, in
fp64, with bounds of what a kernel with fp32 sums and 16-bit operands may be off.
"""

from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24     # half a step of fp32, relative
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}   # half of the least step


def turned(x, positions, frequencies, magnitude, layout, start=0, inverse=False):
    """(values, sum of magnitudes) of x [tokens, heads, head_dim] fp64."""
    x = np.asarray(x, np.float64)
    n = len(frequencies)
    t = np.asarray(positions, np.float64)[:, None, None] * np.asarray(frequencies)
    if inverse:
        t, magnitude = -t, 1.0 / magnitude
    a = x[..., start:start + n] if layout == "half" else x[..., start:start + 2 * n:2]
    b = x[..., start + n:start + 2 * n] if layout == "half" else x[..., start + 1:start + 2 * n:2]
    out, mass = x.copy(), np.abs(x)
    both = np.stack([a * np.cos(t) - b * np.sin(t), b * np.cos(t) + a * np.sin(t)]) * magnitude
    sums = np.stack([np.abs(a) + np.abs(b)] * 2) * magnitude
    for to, v in ((out, both), (mass, sums)):
        if layout == "half":
            to[..., start:start + n], to[..., start + n:start + 2 * n] = v
        else:
            to[..., start:start + 2 * n:2], to[..., start + 1:start + 2 * n:2] = v
    return out, mass


def turned_bound(out, mass, out_type):
    """A sine or cosine is off by 2.2 units of 2^-24 at most (its quarter turn's
    rounding, its series; tests/test_rotary_angles.py derives it and holds them to
    it alone).  Times the magnitude, itself rounded and with `inverse` divided by:
    3 more; two products and their sum: 2 (each value is in one product).  7.2
    units of the sum of magnitudes; 9 leave room for far positions, whose angle
    is rounded in fp64.  Then one rounding to the type."""
    return 9 * U32 * mass + UNIT[out_type] * (np.abs(out) + 9 * U32 * mass) + TINY[out_type]


def gather(rows, table_row, positions):
    """Rows [n, values] of a request's positions; None where there is no block."""
    bs = rows.shape[1]
    out = np.zeros((len(positions), rows.shape[2]))
    there = np.zeros(len(positions), bool)
    for i, p in enumerate(positions):
        b = table_row[p // bs] if 0 <= p and p // bs < len(table_row) else -1
        if 0 <= b < len(rows):
            out[i], there[i] = rows[b, p % bs], True
    return out, there


def attend_one(q, k, v, scale, weight_unit, out_type, chain):
    """One (token, head): q [d] over keys k [n, d], values v [n, dv] in fp64.
    (out, lse, out bound, lse bound).  ``chain``: fp32 additions in a score."""
    if not len(k):
        return np.zeros(v.shape[1]), -np.inf, np.zeros(v.shape[1]), 0.0
    with np.errstate(all="ignore"):
        s = scale * (k @ q)
        top = s.max()
        p = np.exp(s - top)
        l = p.sum()
        o = (p @ v) / l
        mass = (p @ np.abs(v)) / l
    # products of 16-bit values are exact; sums in fp32, the scaling, the
    # exponential's argument and result
    mag = abs(scale) * (np.abs(k) @ np.abs(q)).max()
    ds = mag * (chain + 8) * 2 * U32 + np.abs(s).max() * 6 * U32
    rel = 2 * ds + (len(k) + 64) * 2 * U32 + weight_unit
    lse = top + np.log(l)
    bound = mass * rel + UNIT[out_type] * (np.abs(o) + mass * rel) + TINY[out_type]
    # fp16 weights are whole multiples of 2^-24 of 2^13 times them
    bound += len(k) * np.abs(v).max() * 2.0 ** -37 / l
    return o, lse, bound, ds + (len(k) + 64) * 2 * U32 + abs(lse) * 4 * U32


def attend(q, rows, rank, ctx, new, table, scale, window=0, out_type="bf16", heads_of=None):
    """Absorbed attention; q [tokens, heads, rank + rope], rows [blocks,
    block_tokens, rank + rope], values of the 16-bit types.  (out, lse, bounds)."""
    q = np.asarray(q, np.float64)
    tokens, heads, d = q.shape
    out, lse = np.zeros((tokens, heads, rank)), np.full((tokens, heads), -np.inf)
    ob, lb = np.zeros_like(out), np.zeros_like(lse)
    row = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        keys, there = gather(rows, table[r], range(c + n)) if n else (None, None)
        for i in range(n):
            see = there & (np.arange(c + n) <= c + i)
            if window:
                see &= np.arange(c + n) > c + i - window
            k = keys[see]
            for h in (range(heads) if heads_of is None else heads_of):
                out[row, h], lse[row, h], ob[row, h], lb[row, h] = attend_one(
                    q[row, h], k, k[:, :rank], scale, UNIT[out_type], out_type, d)
            row += 1
    return out, lse, ob, lb


def expand(rows, weight, key_dim, rank, ctx_rows, table, out_type):
    """(k, v, bounds) of ranges [(request, first position, count)]: k [rows,
    heads, key_dim + rope], v [rows, heads, value_dim]."""
    w = np.asarray(weight, np.float64)
    heads = w.shape[0]
    got = np.concatenate([gather(rows, table[r], range(p, p + n))[0] for r, p, n in ctx_rows]
                         + [np.zeros((0, rows.shape[2]))])
    made = np.einsum("rc,hnc->rhn", got[:, :rank], w)
    mass = np.einsum("rc,hnc->rhn", np.abs(got[:, :rank]), np.abs(w))
    turned = np.repeat(got[:, None, rank:], heads, 1)
    # products of 16-bit values are exact; `rank` fp32 additions, one rounding
    off = mass * (rank + 2) * 2 * U32
    bound = off + UNIT[out_type] * (np.abs(made) + off) + TINY[out_type]
    k = np.concatenate([made[..., :key_dim], turned], -1)
    kb = np.concatenate([bound[..., :key_dim], np.zeros_like(turned)], -1)
    return k, made[..., key_dim:], kb, bound[..., key_dim:]


def attend_rows(q, k, v, ctx, new, cu_rows, starts, scale, window=0, out_type="bf16", heads_of=None):
    """(out, lse, bounds) over dense rows."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    tokens, heads, d = q.shape
    out, lse = np.zeros((tokens, heads, v.shape[2])), np.full((tokens, heads), -np.inf)
    ob, lb = np.zeros_like(out), np.zeros_like(lse)
    row = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        a, b = cu_rows[r], cu_rows[r + 1]
        at = starts[r] + np.arange(b - a)
        for i in range(n):
            see = at <= c + i
            if window:
                see &= at > c + i - window
            for h in (range(heads) if heads_of is None else heads_of):
                out[row, h], lse[row, h], ob[row, h], lb[row, h] = attend_one(
                    q[row, h], k[a:b][see, h], v[a:b][see, h], scale, UNIT[out_type], out_type, d)
            row += 1
    return out, lse, ob, lb
