"""Workloads by which rotary positions and latent attention are judged.

Five paths, of sessions whose grafts are mounted at positions of their own:

* ``rotate``: queries or keys turned to their positions, the whole head or a
  part of it, halves or neighbours as pairs, frequencies scaled for long
  contexts;
* ``append``: a step's keys turned on their way into the 8-bit paged cache, the
  values beside them; the touched blocks' tokens read back dense;
* ``latent_append``: one latent and one turned key part a token, into the rows
  of a paged latent cache;
* ``latent_attend``: absorbed attention over that cache, where all heads share
  a token's row: its whole is the key, its latent part the value;
* ``expanded``: a head's own keys and values made from the cached latents, and
  causal attention of prompts over them.

Layouts: key codes [blocks, kv, block_tokens, hd], value codes [blocks, kv, hd,
block_tokens], scales [blocks, kv]; latent rows [blocks, block_tokens, rank +
rope].  The lengths of a case are fixed by the case; the seed deals them to the
requests and makes everything else.
"""

from __future__ import annotations

import math
import zlib
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def _rotate(name, tokens, heads, hd, start, dim, layout, scaling, dtype, far):
    return dict(name=name, op="rotate", tokens=tokens, heads=heads, hd=hd, start=start, dim=dim,
                layout=layout, scaling=scaling, dtype=dtype, far=far)


def _append(name, requests, ctx, new, kv, hd, bs, dim, layout, dtype, out):
    return dict(name=name, op="append", requests=requests, ctx_lo=ctx[0], ctx_hi=ctx[1],
                chunks=requests, new_lo=new[0], new_hi=new[1], kv=kv, hd=hd, bs=bs, dim=dim,
                layout=layout, scaling="none", dtype=dtype, out=out)


def _latent(name, op, requests, ctx, new, rank, rope, bs, dtype, heads=1, chunks=None, window=0,
            nope=0, vd=0, source=""):
    return dict(name=name, op=op, requests=requests, ctx_lo=ctx[0], ctx_hi=ctx[1],
                chunks=requests if chunks is None else chunks, new_lo=new[0], new_hi=new[1],
                rank=rank, rope=rope, bs=bs, dtype=dtype, heads=heads, window=window, nope=nope,
                vd=vd, source=source)


def listed():
    return [
        # A decode step's queries, one token of every session: latency.
        _rotate("rotate_step", 32, 32, 128, 0, 128, "half", "none", "bf16", 8000),
        # A long document's queries far out, the last part of each head turned.
        _rotate("rotate_far_part", 8011, 40, 96, 64, 32, "interleaved", "yarn", "f16", 131_000),
        # A decode step's keys into the 8-bit cache; the open blocks read back.
        _append("append_step_turned", 64, (15, 4000), (1, 1), 8, 128, 64, 128, "half", "bf16",
                "f16"),
        # Grafts mounted at new positions into fresh and half-filled blocks, half a head turned.
        _append("append_grafts_turned", 24, (0, 500), (100, 2000), 4, 256, 32, 128, "interleaved",
                "f16", "bf16"),
        # A decode step's latents of many sessions.
        _latent("latent_append_step", "latent_append", 128, (15, 4000), (1, 1), 256, 32, 16,
                "bf16", source="bf16"),
        # Latent grafts mounted, computed in full precision, kept in 16 bits.
        _latent("latent_append_grafts", "latent_append", 24, (0, 500), (100, 2000), 512, 64, 64,
                "bf16", source="f32"),
        # One chat's next token on a graft of ordinary length: latency.
        _latent("latent_one", "latent_attend", 1, (1021, 1021), (1, 1), 512, 64, 64, "bf16",
                heads=16),
        # An ordinary decode step of the small latent width: sessions of every age.
        _latent("latent_step_ragged", "latent_attend", 32, (190, 8150), (1, 1), 256, 32, 64,
                "bf16", heads=40),
        # A decode step of the large latent width with all its heads.
        _latent("latent_step_heads", "latent_attend", 24, (500, 12_001), (1, 1), 512, 64, 32,
                "bf16", heads=128),
        # A drafted chunk on top of a mounted document, and decoding sessions beside it.
        _latent("latent_mixed", "latent_attend", 9, (700, 7003), (130, 257), 512, 64, 16, "f16",
                heads=16, chunks=1),
        # Fresh prompts of a batch through a head's own keys and values.
        _latent("expanded_prompts", "expanded", 3, (0, 0), (333, 2500), 512, 64, 64, "bf16",
                heads=32, nope=128, vd=128),
        # A chunk of a document behind mounted latents, the small width.
        _latent("expanded_chunk", "expanded", 1, (5011, 5011), (1021, 1021), 256, 32, 32, "f16",
                heads=40, nope=64, vd=64),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotate", "append", "latent_append", "step", "step", "chunk", "expanded"))
    bs = rng.choice((16, 32, 64, 128))
    layout = rng.choice(("half", "interleaved"))
    dtype = rng.choice(("bf16", "f16"))
    rank, rope, heads, nope, vd = rng.choice(((512, 64, 128, 128, 128), (512, 64, 16, 128, 128),
                                              (256, 32, 40, 64, 64), (256, 32, 20, 64, 64)))
    if kind == "rotate":
        hd, start, dim = rng.choice(((128, 0, 128), (256, 0, 64), (192, 128, 64), (96, 64, 32),
                                     (64, 0, 64)))
        n = rng.choice((1, 8, 20, 40))
        c = _rotate("", _spread(rng, 1, 30_000_000 // (n * hd)), n, hd, start, dim, layout,
                    rng.choice(("none", "linear", "yarn")), rng.choice(("bf16", "f16", "f32")),
                    _spread(rng, 100, 1_000_000))
    elif kind == "append":
        kv, hd = rng.choice(((8, 128), (4, 256), (16, 64)))
        n = _spread(rng, 1, 1000)
        c = _append("", max(1, min(64, 15_000 // n, _spread(rng, 1, 64))),
                    (0, _spread(rng, 10, 2000)), (1, n), kv, hd, bs,
                    rng.choice((hd, hd // 2)), layout, rng.choice(("bf16", "f16", "f32")),
                    rng.choice(("f16", "bf16")))
    elif kind == "latent_append":
        n = _spread(rng, 1, 1500)
        c = _latent("", kind, max(1, min(64, 15_000 // n, _spread(rng, 1, 64))),
                    (0, _spread(rng, 10, 2000)), (1, n), rank, rope, bs, dtype,
                    source=rng.choice(("bf16", "f16", "f32")))
    elif kind == "step":
        hi = _spread(rng, 50, 12_000)
        new = rng.choice((1, 1, 1, 2, 3))
        n = max(1, min(_spread(rng, 1, 48), 80_000 // (hi * new)))
        c = _latent("", "latent_attend", n, (max(1, hi // 20), hi), (new, new), rank, rope, bs,
                    dtype, heads=heads, window=rng.choice((0, 0, 0, 700)))
    elif kind == "chunk":
        hi = _spread(rng, 100, 4000)
        n = rng.randint(1, 6)
        c = _latent("", "latent_attend", n, (max(1, hi // 4), hi), (9, _spread(rng, 16, 120)),
                    rank, rope, bs, dtype, heads=min(heads, 40), chunks=1)
    else:
        hi = _spread(rng, 60, 900)
        n = rng.randint(1, 2)
        ctx = rng.choice((0, 0, _spread(rng, 50, 1000)))
        c = _latent("", "expanded", n, (ctx // 2, ctx), (max(1, hi // 5), hi), rank, rope, bs,
                    dtype, heads=min(heads, 32), nope=nope, vd=vd, window=rng.choice((0, 0, 500)))
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(case):
    """Tokens held and tokens new of each request, fixed by the case."""
    text = repr(sorted((k, v) for k, v in case.items() if k != "name"))
    rng = np.random.default_rng(zlib.crc32(text.encode()))

    def some(lo, hi, n):
        x = np.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1), n)) - 1
        return np.clip(np.rint(x), lo, hi).astype(np.int64)

    n = case["requests"]
    ctx = some(case["ctx_lo"], case["ctx_hi"], n)
    new = np.ones(n, np.int64)
    new[:case["chunks"]] = some(case["new_lo"], case["new_hi"], case["chunks"])
    if n > 1:  # the longest is there whatever the draw
        ctx[0] = case["ctx_hi"]
        new[0] = case["new_hi"] if case["chunks"] else 1
    return ctx, new


def _blocks(n, bs):
    return -(-n // bs)


# Frequencies (a position's angle) of a case's pairs and what the turned values
# are multiplied by, in 64 bits.
BASE, FACTOR, TRAINED, FAST, SLOW = 10_000.0, 8.0, 4096, 32.0, 1.0


def _frequencies(dim, scaling):
    """``linear``: all positions divided by FACTOR.  ``yarn``: frequencies that
    turn more than FAST times in TRAINED positions stay, those that turn less
    than SLOW times are divided, between them a ramp over the pair's number;
    the values grow by 0.1 ln FACTOR + 1."""
    f = BASE ** (-2.0 * np.arange(dim // 2) / dim)
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling == "yarn":
        at = lambda turns: dim * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
        low, high = max(math.floor(at(FAST)), 0), min(math.ceil(at(SLOW)), dim - 1)
        ramp = np.clip((np.arange(dim // 2) - low) / max(high - low, 0.001), 0, 1)
        return f / FACTOR * ramp + f * (1 - ramp), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


def _codes(gen, shape):
    """Codes of normal values, a block's largest near 127."""
    x = torch.randn(shape, generator=gen, device=DEV)
    return x.mul_(33.0).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV)  # noqa: E731
    s = SimpleNamespace(case=case)
    if op == "rotate":
        n = case["tokens"]
        # a step's sessions stand anywhere, prompts' positions follow each other
        first = rng.integers(0, max(1, case["far"] - n), n if n < 200 else n // 200)
        at = np.concatenate([f + np.arange(-(-n // len(first))) for f in first])[:n]
        s.positions = torch.from_numpy(at.astype(np.int32)).to(DEV)
        s.x = (normal(n, case["heads"], case["hd"]) * 1.5).to(dt)
        dim = case["dim"]
    else:
        bs = case["bs"]
        ctx, new = _lengths(case)
        deal = rng.permutation(len(ctx))
        ctx, new = ctx[deal], new[deal]
        total = _blocks(ctx + new, bs)
        pool = int(total.sum()) + 8
        s.ctx_h, s.new_h, s.bs, s.tokens = ctx, new, bs, int(new.sum())
        s.width, s.max_new = int(total.max()) + 1, int(new.max())
        ids = torch.from_numpy(rng.permutation(pool).astype(np.int32))
        table = torch.full((len(ctx), s.width), -1, dtype=torch.int32)
        mine = torch.arange(s.width)[None, :] < torch.from_numpy(total)[:, None]
        table[mine] = ids[:int(total.sum())]
        s.table = table.to(DEV)
        s.ctx = torch.from_numpy(ctx.astype(np.int32)).to(DEV)
        s.new = torch.from_numpy(new.astype(np.int32)).to(DEV)
        cu = lambda n: torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).to(DEV)  # noqa: E731
        s.cu = cu(new)
        spare = ids[int(total.sum()):].long().to(DEV)   # blocks of nobody hold anything
        dim = case["dim"] if op == "append" else case["rope"]
    if op == "append":
        kv, hd = case["kv"], case["hd"]
        s.k_codes = _codes(gen, (pool, kv, bs, hd))
        s.v_codes = _codes(gen, (pool, kv, hd, bs))
        s.k_scales, s.v_scales = (torch.exp(0.3 * normal(pool, kv)) / 36.0 for _ in "kv")
        s.k_scales[spare] = float("nan")
        s.v_scales[spare] = float("nan")
        # channels of unlike size, as keys have them
        s.k = (normal(s.tokens, kv, hd) * torch.exp(0.5 * normal(kv, hd))).to(dt)
        s.v = normal(s.tokens, kv, hd).to(dt)
        s.out = DTYPES[case["out"]]
        s.start_h = ctx // bs * bs
        rows = ctx + new - s.start_h
        s.n_rows, s.touched = int(rows.sum()), int((total - ctx // bs).sum())
        s.start, s.cu_rows = torch.from_numpy(s.start_h.astype(np.int32)).to(DEV), cu(rows)
    elif op != "rotate":
        rank, rope, heads = case["rank"], case["rope"], case["heads"]
        # latents after their norm, channels of unlike size
        s.rows = (normal(pool, bs, rank + rope)
                  * torch.exp(0.3 * normal(rank + rope))).to(dt)
        s.rows[spare] = float("nan")
        s.freq, s.magnitude = _frequencies(rope, "yarn")
    if op == "latent_append":
        source = DTYPES[case["source"]]
        s.latent, s.rope_key = normal(s.tokens, rank).to(source), normal(s.tokens, rope).to(source)
    if op == "latent_attend":
        s.q = (normal(s.tokens, heads, rank + rope) * 0.7).to(dt)
        s.scale = 1.0 / math.sqrt(192 if rank == 512 else 96)
    if op == "expanded":
        s.q = normal(s.tokens, heads, case["nope"] + rope).to(dt)
        s.weight = (normal(heads, case["nope"] + case["vd"], rank) / math.sqrt(rank)).to(dt)
        s.scale = 1.0 / math.sqrt(case["nope"] + rope)
        s.n_rows = int((ctx + new).sum())
        s.start, s.cu_rows = torch.zeros_like(s.ctx), cu(ctx + new)
    if op in ("rotate", "append"):
        s.freq, s.magnitude = _frequencies(dim, case["scaling"])
    if own:
        from graftrepository_amd import KvBatch, KvCache, LatentCache, Rotary
        scaling = "yarn" if op == "latent_append" else case.get("scaling", "none")
        more = dict(factor=FACTOR, trained=TRAINED, fast=FAST, slow=SLOW) if scaling == "yarn" else \
            dict(factor=FACTOR) if scaling == "linear" else {}
        s.rotary = Rotary(dim, base=BASE, layout=case.get("layout", "interleaved"),
                          scaling=None if scaling == "none" else scaling, **more)
        if op != "rotate":
            s.batch = KvBatch(s.ctx, s.new, s.table, bs, tokens=s.tokens, max_new=s.max_new,
                              heads=case.get("heads", case.get("kv")),
                              kv_heads=case.get("kv", 1), window=case.get("window", 0),
                              latent=op in ("latent_attend", "expanded"))
            s.batch.plan()   # once a step; every layer's calls share it
            s.cache = KvCache(s.k_codes, s.v_codes, s.k_scales, s.v_scales) if op == "append" \
                else LatentCache(s.rows, rank)
    s.freq = torch.from_numpy(s.freq).to(DEV) if op != "latent_attend" and op != "expanded" else None
    return s


# ------------------------------------------------------------- plain forms

def _turn(x, positions, freq, magnitude, layout, start=0):
    """x [tokens, heads, hd] in 32 bits, channels from `start` on turned; the
    angles in 64 bits."""
    dim = 2 * freq.numel()
    t = positions.double()[:, None] * freq
    cos, sin = ((f(t) * magnitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    part = x[..., start:start + dim]
    if layout == "half":
        a, b = part[..., :dim // 2], part[..., dim // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([x[..., :start], turned, x[..., start + dim:]], -1)


def _plain_rotate(s):
    c = s.case
    return _turn(s.x.float(), s.positions, s.freq, s.magnitude, c["layout"], c["start"]).to(s.x.dtype)


def _token_rows(s):
    """Request, position, physical block and place in it of every new token."""
    i = torch.arange(s.tokens, device=DEV)
    r = torch.searchsorted(s.cu[1:], i, right=True)
    pos = s.ctx.long()[r] + i - s.cu.long()[r]
    return r, pos, s.table[r, pos // s.bs].long(), pos % s.bs


def _plain_write(x, codes, scales, transposed, tok, blocks, kept):
    """Quantise x [tokens, kv, hd] into `codes`, block by block."""
    block, place = tok
    top = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(-1), "amax")[blocks]
    old = torch.where(kept.amax(-1)[:, None], scales[blocks], torch.zeros_like(top))
    scale = torch.maximum(old, top / 127.0)
    scales[blocks] = scale
    ratio = torch.where(scale > 0, old / scale, torch.zeros_like(scale))[:, :, None, None]
    before = codes[blocks]
    stay = kept[:, None, None, :] if transposed else kept[:, None, :, None]
    codes[blocks] = torch.where(stay, (before.float() * ratio).round().to(torch.int8), before)
    each = scales[block][:, :, None]
    q = torch.where(each > 0, (x / each).round().clamp(-127, 127), torch.zeros_like(x)).to(torch.int8)
    if transposed:
        codes.permute(0, 3, 1, 2)[block, place] = q
    else:
        codes.permute(0, 2, 1, 3)[block, place] = q


def _row_places(s):
    """Physical block and place of every row that is read back."""
    i = torch.arange(s.n_rows, device=DEV)
    r = torch.searchsorted(s.cu_rows[1:], i, right=True)
    pos = s.start.long()[r] + i - s.cu_rows.long()[r]
    return s.table[r, pos // s.bs].long(), pos % s.bs


def _plain_append(s):
    bs = s.bs
    _, pos, block, place = _token_rows(s)
    ctx, new = s.ctx.long(), s.new.long()
    first = ctx // bs
    count = (ctx + new + bs - 1) // bs - first
    r = torch.repeat_interleave(torch.arange(len(ctx), device=DEV), count, output_size=s.touched)
    j = torch.arange(s.touched, device=DEV) - (count.cumsum(0) - count)[r] + first[r]
    blocks = s.table[r, j].long()
    kept = (j * bs)[:, None] + torch.arange(bs, device=DEV)[None, :] < ctx[r][:, None]
    k = _turn(s.k.float(), pos, s.freq, s.magnitude, s.case["layout"])
    _plain_write(k, s.k_codes, s.k_scales, False, (block, place), blocks, kept)
    _plain_write(s.v.float(), s.v_codes, s.v_scales, True, (block, place), blocks, kept)
    block, place = _row_places(s)
    k = s.k_codes.permute(0, 2, 1, 3)[block, place].float() * s.k_scales[block][:, :, None]
    v = s.v_codes.permute(0, 3, 1, 2)[block, place].float() * s.v_scales[block][:, :, None]
    return dict(k=k.to(s.out), v=v.to(s.out), k_scales=s.k_scales, v_scales=s.v_scales)


def _plain_latent_append(s):
    _, pos, block, place = _token_rows(s)
    turned = _turn(s.rope_key.float()[:, None], pos, s.freq, s.magnitude, "interleaved")[:, 0]
    s.rows[block, place] = torch.cat([s.latent.float(), turned], -1).to(s.rows.dtype)
    return s.rows


def _softmax_rows(s, q, k, v, keys):
    """q [R, H, N, d] against k [R, H or 1, L, d], v alike; keys [R]: how many
    there are.  Causal by position, within the window; o [R, H, N, dv], lse."""
    n_req, heads, n, d = q.shape
    j = torch.arange(k.shape[2], device=DEV)
    pos = s.ctx.long()[:, None] + torch.arange(n, device=DEV)
    see = (j[None, None, :] <= pos[:, :, None]) & (j[None, None, :] < keys[:, None, None])
    if s.case["window"]:
        see = see & (j[None, None, :] > pos[:, :, None] - s.case["window"])
    # where heads share their keys, all of them are rows of one product
    q = q.reshape(n_req, k.shape[1], -1, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s.scale)
    score = score.view(n_req, heads, n, -1).masked_fill_(~see[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_req, k.shape[1], -1, k.shape[2]), v).view(n_req, heads, n, -1)
    return torch.where(total > 0, o / total, torch.zeros_like(o)), (top + torch.log(total))[..., 0]


def _padded_queries(s):
    """The step's queries as [R, H, N, d] in 32 bits, and how to take [R, H,
    N, ...] back to its rows."""
    i = torch.arange(s.max_new, device=DEV)
    row = (s.cu.long()[:-1, None] + i).clamp(max=s.tokens - 1)
    r, pos, _, _ = _token_rows(s)
    n = pos - s.ctx.long()[r]
    return s.q.float()[row].transpose(1, 2).contiguous(), lambda x: x.transpose(1, 2)[r, n]


def _plain_latent_attend(s):
    keys = s.ctx.long() + s.new.long()
    k = s.rows[s.table.long().clamp(min=0)].float().view(len(s.ctx_h), 1, s.width * s.bs, -1)
    there = torch.arange(s.width * s.bs, device=DEV)[None, :] < keys[:, None]
    k = torch.where(there[:, None, :, None], k, torch.zeros((), device=DEV))
    q, back = _padded_queries(s)
    o, lse = _softmax_rows(s, q, k, k[..., :s.case["rank"]].contiguous(), keys)
    return dict(out=back(o).to(s.q.dtype), lse=back(lse))


def _plain_expanded(s):
    c = s.case
    rank, heads, nope = c["rank"], c["heads"], c["nope"]
    block, place = _row_places(s)
    row = s.rows[block, place].float()
    made = (row[:, :rank] @ s.weight.float().view(-1, rank).t()).view(s.n_rows, heads, -1)
    turned = row[:, None, rank:].expand(-1, heads, -1)
    k = torch.cat([made[..., :nope], turned], -1).to(s.rows.dtype)
    v = made[..., nope:].to(s.rows.dtype).contiguous()
    # attention takes what was kept of them
    keys = s.ctx.long() + s.new.long()
    longest = int((s.ctx_h + s.new_h).max())
    at = s.cu_rows.long()[:-1, None] + torch.arange(longest, device=DEV)
    there = (torch.arange(longest, device=DEV)[None, :] < keys[:, None])[:, None, :, None]
    at = at.clamp(max=s.n_rows - 1)
    pk, pv = (torch.where(there, x[at].float().transpose(1, 2), torch.zeros((), device=DEV)).contiguous()
              for x in (k, v))
    q, back = _padded_queries(s)
    o, lse = _softmax_rows(s, q, pk, pv, keys)
    return dict(k=k, v=v, out=back(o).to(s.q.dtype), lse=back(lse))


def run(s):
    c, op = s.case, s.case["op"]
    if not own:
        return {"rotate": _plain_rotate, "append": _plain_append,
                "latent_append": _plain_latent_append, "latent_attend": _plain_latent_attend,
                "expanded": _plain_expanded}[op](s)
    if op == "rotate":
        return s.rotary.apply(s.x, s.positions, start=c["start"])
    if op == "append":
        s.cache.append(s.batch, s.k, s.v, rotary=s.rotary)
        k, v = s.cache.read(s.table, s.start, s.cu_rows, s.n_rows, dtype=s.out)
        return dict(k=k, v=v, k_scales=s.k_scales, v_scales=s.v_scales)
    if op == "latent_append":
        s.cache.append(s.batch, s.latent, s.rope_key, rotary=s.rotary)
        return s.rows
    if op == "latent_attend":
        out, lse = s.cache.attend(s.batch, s.q, s.scale, return_lse=True)
        return dict(out=out, lse=lse)
    from graftrepository_amd import attend_rows
    k, v = s.cache.expand(s.weight, s.case["nope"], s.table, s.start, s.cu_rows, s.n_rows)
    out, lse = attend_rows(s.batch, s.q, k, v, s.cu_rows, softmax_scale=s.scale, return_lse=True)
    return dict(k=k, v=v, out=out, lse=lse)


# ------------------------------------------------------- 64-bit definition

def _exact_turn(x, positions, freq, magnitude, layout):
    """Pairs as complex numbers, times e^(i angle)."""
    t = positions.double()[:, None, None] * freq
    z = torch.polar(torch.full_like(t, magnitude), t)
    x = x.double()
    n = freq.numel()
    pairs = torch.stack([x[..., :n], x[..., n:]], -1) if layout == "half" else x.view(*x.shape[:-1], n, 2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    return torch.cat([y[..., 0], y[..., 1]], -1) if layout == "half" else y.flatten(-2)


def _exact_heads(q, k, v, ctx, scale, window):
    """One request: q [n, H, d], k and v one head's [m, d] each by `h`."""
    n, heads, _ = q.shape
    m = k(0).shape[0]
    i = torch.arange(ctx, ctx + n, device=DEV)[:, None]
    j = torch.arange(m, device=DEV)[None, :]
    hide = (j > i) | ((j <= i - window) if window else (j < 0))
    o, lse = [], []
    for h in range(heads):
        sc = ((q[:, h] @ k(h).T) * scale).masked_fill(hide, -math.inf)
        lse.append(torch.logsumexp(sc, -1))
        o.append(torch.exp(sc - lse[-1][:, None]) @ v(h))
    return torch.stack(o, 1), torch.stack(lse, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotate":
        x, a, b = s.x.double(), case["start"], case["start"] + case["dim"]
        x[..., a:b] = _exact_turn(x[..., a:b], s.positions, s.freq, s.magnitude, case["layout"])
        return x
    bs = s.bs
    each = list(zip(s.ctx_h.tolist(), s.new_h.tolist(), s.cu.tolist()))
    if op == "latent_append":
        rows, rank = s.rows.double(), case["rank"]
        for r, (ctx, new, at) in enumerate(each):
            p = torch.arange(ctx, ctx + new, device=DEV)
            key = _exact_turn(s.rope_key[at:at + new, None], p, s.freq, s.magnitude, "interleaved")
            rows[s.table[r, p // bs].long(), p % bs] = torch.cat(
                [s.latent[at:at + new].double(), key[:, 0]], -1)
        return rows
    if op == "latent_attend":
        rank, parts = case["rank"], []
        for r, (ctx, new, at) in enumerate(each):
            k = s.rows[s.table[r, :_blocks(ctx + new, bs)].long()].double().flatten(0, 1)[:ctx + new]
            parts.append(_exact_heads(s.q[at:at + new].double(), lambda h: k, lambda h: k[:, :rank],
                                      ctx, s.scale, case["window"]))
        return dict(out=torch.cat([p[0] for p in parts]), lse=torch.cat([p[1] for p in parts]))
    if op == "expanded":
        rank, nope, heads = case["rank"], case["nope"], case["heads"]
        w, keys, values, parts = s.weight.double(), [], [], []
        for r, (ctx, new, at) in enumerate(each):
            c = s.rows[s.table[r, :_blocks(ctx + new, bs)].long()].double().flatten(0, 1)[:ctx + new]
            k = [torch.cat([c[:, :rank] @ w[h, :nope].T, c[:, rank:]], -1) for h in range(heads)]
            v = [c[:, :rank] @ w[h, nope:].T for h in range(heads)]
            keys.append(torch.stack(k, 1))
            values.append(torch.stack(v, 1))
            # attention's inputs are what was kept of them
            low = lambda x: x.to(s.rows.dtype).double()  # noqa: E731
            parts.append(_exact_heads(s.q[at:at + new].double(), lambda h: low(k[h]),
                                      lambda h: low(v[h]), ctx, s.scale, case["window"]))
        return dict(k=torch.cat(keys), v=torch.cat(values), out=torch.cat([p[0] for p in parts]),
                    lse=torch.cat([p[1] for p in parts]))
    scales = {"k": s.k_scales.double(), "v": s.v_scales.double()}
    codes = {"k": s.k_codes.double(), "v": s.v_codes.double().transpose(2, 3)}
    rows = {"k": [], "v": []}
    dim, kv, hd = case["dim"], case["kv"], case["hd"]
    for r, (ctx, new, at) in enumerate(each):
        ids = s.table[r, ctx // bs:_blocks(ctx + new, bs)].long()
        tail = ctx % bs
        k = s.k[at:at + new].double()
        k[..., :dim] = _exact_turn(k[..., :dim], torch.arange(ctx, ctx + new, device=DEV), s.freq,
                                   s.magnitude, case["layout"])
        for name, x in (("k", k), ("v", s.v[at:at + new].double())):
            pad = len(ids) * bs - tail - new
            y = torch.cat([x.new_zeros(tail, kv, hd), x, x.new_zeros(pad, kv, hd)])
            y = y.view(len(ids), bs, kv, hd)
            scale = y.abs().amax((1, 3)) / 127
            if tail:
                scale[0] = torch.maximum(scale[0], scales[name][ids[0]])
            q = torch.round(y / scale[:, None, :, None]).clamp(-127, 127)
            if tail:
                old = codes[name][ids[0]].transpose(0, 1)[:tail]
                q[0, :tail] = torch.round(old * (scales[name][ids[0]] / scale[0])[None, :, None])
            scales[name][ids] = scale
            rows[name].append((q * scale[:, None, :, None]).reshape(-1, kv, hd)[:tail + new])
    return dict(k=torch.cat(rows["k"]), v=torch.cat(rows["v"]), k_scales=scales["k"],
                v_scales=scales["v"])


# ------------------------------------------------------------ least work

def _pairs(ctx, new, window):
    """(token, key) pairs that are seen, and keys that some token sees."""
    pairs = 0
    for c, n in zip(ctx.tolist(), new.tolist()):
        see = np.arange(c + 1, c + n + 1)
        pairs += int((np.minimum(see, window) if window else see).sum())
    first = np.maximum(ctx + 1 - window, 0) if window else np.zeros_like(ctx)
    return pairs, int((ctx + new - first).sum())


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["hd"] * size + 4 * case["tokens"], "flops": 3 * n * case["dim"]}
    ctx, new = _lengths(case)
    bs, n_tok = case["bs"], int(new.sum())
    if case["op"] == "append":
        kv, hd = case["kv"], case["hd"]
        back = int((ctx + new - ctx // bs * bs).sum())
        touched = int((_blocks(ctx + new, bs) - ctx // bs).sum())
        values = n_tok * (size + 1) + (back - n_tok) + back * SIZES[case["out"]]
        return {"bytes": 2 * kv * hd * values + 8 * kv * touched,
                "flops": (4 * 2 * hd + 3 * case["dim"]) * kv * n_tok}
    rank, rope, heads = case["rank"], case["rope"], case["heads"]
    if case["op"] == "latent_append":
        return {"bytes": n_tok * (rank + rope) * (SIZES[case["source"]] + size),
                "flops": 3 * rope * n_tok}
    pairs, seen = _pairs(ctx, new, case["window"])
    if case["op"] == "latent_attend":
        return {"bytes": seen * (rank + rope) * size
                + heads * n_tok * ((2 * rank + rope) * size + 4),
                "flops": 2 * pairs * heads * (2 * rank + rope)}
    rows, nope, vd = int((ctx + new).sum()), case["nope"], case["vd"]
    made = rows * heads * (nope + rope + vd) * size
    return {"bytes": rows * (rank + rope) * size + heads * (nope + vd) * rank * size + 2 * made
            + n_tok * heads * ((nope + rope + vd) * size + 4),
            "flops": 2 * rows * heads * (nope + vd) * rank + 2 * pairs * heads * (nope + rope + vd)}
