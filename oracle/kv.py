"""The 8-bit key/value cache's laws on the host, in numpy.

``plan`` is whole numbers.  ``append`` is the law's fp32 arithmetic (its
divisions, products and roundings are IEEE single operations, so numpy
reproduces them bit for bit); ``read`` likewise.  ``attend`` is computed in
fp64, with ``attend_bound``: how far a kernel with fp32 sums (and, where
``half_p``, probabilities rounded to fp16) may be from it.
"""

from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24     # half an ulp of fp32, relative
OUT_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def plan(ctx, new, table, bs, tokens, free=None, head=0):
    """(table, cu, slots, positions, head) of a step."""
    table = np.array(table, np.int32)
    width = table.shape[1]
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    slots = np.full(tokens, -1, np.int64)
    positions = np.full(tokens, -1, np.int32)
    at = head
    for r, (c, n) in enumerate(zip(ctx, new)):
        held, total = -(-c // bs), -(-(c + n) // bs)
        if free is not None and n > 0:
            for j in range(held, min(total, width)):
                table[r, j] = free[at] if at < len(free) else -1
                at += 1
        for i in range(n):
            p = c + i
            b = table[r, p // bs] if p // bs < width else -1
            positions[cu[r] + i] = p
            slots[cu[r] + i] = b * bs + p % bs if b >= 0 else -1
    return table, cu, slots, positions, min(at, len(free)) if free is not None else head


def append(codes, scales, x, ctx, new, table, transposed):
    """Quantise x fp32 [tokens, kv, hd] in place; `codes` [blocks, kv, bs,
    hd], or [blocks, kv, hd, bs] where `transposed`."""
    view = codes.transpose(0, 1, 3, 2) if transposed else codes
    bs = view.shape[2]
    f = np.float32
    row = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        p = c
        while p < c + n:
            place = p % bs
            count = min(bs - place, c + n - p)
            j = p // bs
            b = table[r, j] if j < table.shape[1] else -1
            part = x[row:row + count]                           # [count, kv, hd]
            row, p = row + count, p + count
            if b < 0:
                continue
            with np.errstate(all="ignore"):
                for g in range(view.shape[1]):
                    y = part[:, g].astype(f)
                    old = scales[b, g] if place else f(0)
                    scale = np.maximum(old, np.abs(y).max() * (f(1) / f(127)))
                    if not np.isfinite(y).all() or not np.isfinite(old):
                        scale = f(np.nan)
                    if place and not scale == old:
                        ratio = old / scale if scale > 0 else f(0)
                        kept = view[b, g, :place]
                        view[b, g, :place] = np.rint(kept.astype(f) * f(ratio)).astype(np.int8)
                    q = np.clip(np.rint(y / scale), -127, 127) if scale > 0 else np.zeros_like(y)
                    view[b, g, place:place + count] = q.astype(np.int8)
                    scales[b, g] = scale


def values(codes, scales, blocks, transposed):
    """fp32 values [tokens, kv, hd] of physical blocks in order; blocks below
    0 read as 0."""
    view = codes.transpose(0, 1, 3, 2) if transposed else codes
    _, kv, bs, hd = view.shape
    out = np.zeros((len(blocks), bs, kv, hd), np.float32)
    for i, b in enumerate(blocks):
        if b >= 0:
            with np.errstate(invalid="ignore"):    # a scale that is no number
                out[i] = (view[b].astype(np.float32) * scales[b][:, None, None]).transpose(1, 0, 2)
    return out.reshape(len(blocks) * bs, kv, hd)


def attend(q, k_codes, v_codes, k_scales, v_scales, ctx, new, table, scale, window=0,
           out_type="f32", half_p=True):
    """(out, lse, out_bound, lse_bound) in fp64; q [tokens, heads, hd] holds
    the values of the kernel's input type."""
    q = np.asarray(q, np.float64)
    tokens, heads, hd = q.shape
    kv, bs = k_codes.shape[1], k_codes.shape[2]
    group = heads // kv
    out = np.zeros((tokens, heads, hd))
    lse = np.full((tokens, heads), -np.inf)
    ob, lb = np.zeros_like(out), np.zeros_like(lse)
    row = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        total = c + n
        blocks = [int(table[r, j]) if j < table.shape[1] else -1 for j in range(-(-total // bs))]
        if n and blocks:
            kd = values(k_codes, k_scales, blocks, False)[:total].astype(np.float64)
            vd = values(v_codes, v_scales, blocks, True)[:total].astype(np.float64)
            there = np.repeat(np.array(blocks) >= 0, bs)[:total]
        for i in range(n):
            pos = c + i
            see = there & (np.arange(total) <= pos)
            if window:
                see &= np.arange(total) > pos - window
            idx = np.nonzero(see)[0]
            if len(idx):
                for h in range(heads):
                    g = h // group
                    kk, vv = kd[idx, g], vd[idx, g]
                    qq = q[row + i, h]
                    with np.errstate(all="ignore"):
                        s = scale * (kk @ qq)
                        top = s.max()
                        p = np.exp(s - top)
                        l = p.sum()
                        o = (p @ vv) / l
                        mass = (p @ np.abs(vv)) / l
                    out[row + i, h] = o
                    lse[row + i, h] = top + np.log(l)
                    # a score: hd products and sums in fp32 (an error of one
                    # unit each against the sum of magnitudes), the query's
                    # own 22 bits, code * scale, the scalings; its exp takes
                    # that as a relative error, twice (numerator, sum)
                    mag = abs(scale) * (np.abs(kk) @ np.abs(qq)).max() \
                        + abs(scale) * np.abs(qq).max() * np.abs(kk).sum(1).max() * 2.0 ** -4
                    ds = mag * (hd + 16) * 2 * U32 + np.abs(s).max() * 4 * U32
                    rel = 2 * ds + (len(idx) + 32) * 2 * U32
                    rel += 2.0 ** -11 if half_p else 2.0 ** -20
                    ob[row + i, h] = mass * rel + np.abs(o) * OUT_UNIT[out_type] + 2.0 ** -24 * (
                        out_type == "f16")
                    # what underflows: exp in fp32; the fp16 probabilities
                    # (scaled by 2^15 and by the largest value scale) are
                    # whole multiples of 2^-24
                    ob[row + i, h] += len(idx) * np.abs(vv).max() * (
                        2.0 ** -38 if half_p else 2.0 ** -52) / l
                    lb[row + i, h] = ds + (len(idx) + 32) * 2 * U32 + abs(lse[row + i, h]) * 4 * U32
        row += n
    return out, lse, ob, lb
