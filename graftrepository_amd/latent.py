"""A paged cache of latent vectors, for models whose keys and values come from
one (the MLA dialect's).

A row holds a token's latent and its turned key part, shared by all heads::

    batch = KvBatch(..., heads=40, kv_heads=1, latent=True)
    batch.plan()                                           # once per step
    cache.append(batch, latent, key_part, rotary=rotary)   # per layer
    out = cache.attend(batch, q, scale)                    # per layer, absorbed
    rows = cache.read(table, starts, cu_rows, rows)        # dense, to harvest

In the absorbed form a head's query is taken to the latent's space before (its
own part times the weights that make a head's keys), and its output, a mean of
latents, goes through the weights that make its values after.  Prompts take less
in the expanded form::

    k, v = cache.expand(weight, key_dim, table, starts, cu_rows, rows)
    out = attend_rows(batch, q, k, v, cu_rows)

Batches, memory, streams and errors are those of ``kv_cache``; laws and layouts
those of ``include/grm_hip_router.h``.
"""

from __future__ import annotations

import ctypes
import math
import sys

from . import _lib
from .kv_cache import (KvBatch, _call, _copied, _dense, _empty, _is_torch, _name_of,
                       _no_gradient, _off, _one_device, _rows, _same_device, _stream,
                       _torch_stream, _type, i32, u64, vp)
from .payload import DeviceArray


class _LatentDesc(ctypes.Structure):
    _fields_ = [("rows", vp), ("blocks", u64), ("block_tokens", i32), ("rank", i32),
                ("rope", i32), ("dtype", i32)]


def _flat(a, what: str, tokens: int, values: int):
    """(address, type, row stride) of [tokens, values] rows."""
    if len(a.shape) != 2:
        raise ValueError(f"{what} must have shape {(tokens, values)}, got {tuple(a.shape)}")
    if isinstance(a, DeviceArray):
        name = _type(a, what)
        if name not in ("f32", "bf16", "f16"):
            raise ValueError(f"{what} must be f32, bf16 or f16, got {a.dtype}")
        if tuple(a.shape) != (tokens, values):
            raise ValueError(f"{what} must have shape {(tokens, values)}, got {tuple(a.shape)}")
        return a.data_ptr(), name, values
    if not hasattr(a, "unsqueeze"):
        _type(a, what)
    ptr, name, stride, _ = _rows(a.unsqueeze(1), what, (tokens, 1, values))
    return ptr, name, stride


def _latent_batch(batch: KvBatch) -> None:
    if batch._latent is None:
        raise ValueError("the batch has no latent schedule: make it with latent=True")


def _aligned(a, what: str, shape, dtype: str, stream):
    """(the values, their (address, row stride, head stride)), copied where a
    torch tensor's rows are not 16-byte aligned."""
    row = _rows(a, what, shape)
    if row[1] != dtype:
        raise ValueError(f"{what} must be {dtype}, got {a.dtype}")
    if _off(row) and _is_torch(a):
        a = _copied(a, stream)
        row = _rows(a, what, shape)
    return a, (row[0], row[2], row[3])


def _output(like, out, shape, dtype: str, device: int, stream):
    """(the output, its (address, row stride, head stride), what it is copied
    from where its own rows are not 16-byte aligned)."""
    if out is None:
        out = _empty(like, shape, dtype, stream)
        return out, (out.data_ptr(), shape[1] * shape[2], shape[2]), None
    _same_device(out, "out", device)
    result, row = _aligned(out, "out", shape, dtype, stream)  # rows that are not written stay
    return out, row, None if result is out else result


def _statistics(like, lse, wanted: bool, shape, device: int, stream):
    if lse is None:
        if not wanted:
            return None, None
        lse = _empty(like, shape, "f32", stream)
        return lse, lse.data_ptr()
    at = _dense(lse, "lse", "f32", shape)
    _same_device(lse, "lse", device)
    return lse, at


def _written(out, result, on: int) -> None:
    if result is not None:
        with sys.modules["torch"].cuda.stream(_torch_stream(out, on)):
            out.copy_(result)


class LatentCache:
    """The latent cache of one layer, over the caller's ``rows`` [blocks,
    block_tokens, rank + rope] (bf16 or f16), of which ``rank`` values are the
    latent and the rest the key part.  ``LatentCache.empty`` allocates them."""

    def __init__(self, rows, rank: int):
        self._lib = _lib.load()
        if len(rows.shape) != 3:
            raise ValueError("rows must be [blocks, block_tokens, rank + rope]")
        blocks, bs, values = (int(n) for n in rows.shape)
        rank = int(rank)
        name = _type(rows, "rows")
        if name not in ("bf16", "f16"):
            raise ValueError(f"rows must be bf16 or f16, got {rows.dtype}")
        d = self._desc = _LatentDesc()
        d.rows = _dense(rows, "rows", name, (blocks, bs, values))
        if bs not in (16, 32, 64, 128):
            raise ValueError("block_tokens must be 16, 32, 64 or 128")
        if rank % 16 or not 0 < rank <= 512:
            raise ValueError("rank must be a multiple of 16, at most 512")
        rope = values - rank
        if rope % 16 or not 0 <= rope <= 128:
            raise ValueError("rope must be a multiple of 16, at most 128")
        self.device = _one_device(rows=rows)
        d.blocks, d.block_tokens, d.rank, d.rope = blocks, bs, rank, rope
        d.dtype = _lib.DTYPE_CODES[name]
        self.rows, self.dtype = rows, name
        self.blocks, self.block_tokens, self.rank, self.rope = blocks, bs, rank, rope
        self._ref = ctypes.byref(d)

    @classmethod
    def empty(cls, blocks: int, block_tokens: int, rank: int, rope: int,
              dtype: str = "f16") -> "LatentCache":
        """A cache in memory of its own (a DeviceArray), contents undefined:
        every row is written before it is read."""
        from .kv_cache import _NUMPY
        if dtype not in ("bf16", "f16"):
            raise ValueError("rows are bf16 or f16")
        return cls(DeviceArray((blocks, block_tokens, rank + rope), _NUMPY[dtype]), rank)

    def append(self, batch: KvBatch, latent, key_part=None, stream=None, *, rotary=None) -> None:
        """The step's ``latent`` [tokens, rank] and ``key_part`` [tokens, rope]
        (f32, bf16 or f16, of one type; any row strides) into their rows,
        rounded once; with a ``Rotary`` the key part's first channels are turned
        to the batch's positions on the way."""
        batch._ready_for(self)
        tokens = batch._desc.tokens
        lp, name, lt = _flat(latent, "latent", tokens, self.rank)
        kp, kt = None, 0
        if self.rope:
            if key_part is None:
                raise ValueError("the cache's rows have a key part")
            kp, kname, kt = _flat(key_part, "key_part", tokens, self.rope)
            if kname != name:
                raise ValueError("latent and key_part must have one type")
            _same_device(key_part, "key_part", self.device)
        elif key_part is not None or rotary is not None:
            raise ValueError("the cache's rows have no key part")
        _same_device(latent, "latent", self.device)
        rc = _call(self._lib.grm_hip_latent_append, latent, self.device, self._ref, batch._ref,
                   rotary._ref if rotary is not None else None, lp, kp, _lib.DTYPE_CODES[name], lt,
                   kt, batch._on(latent, stream))
        if rc:
            _lib.check(rc, "latent append")

    def attend(self, batch: KvBatch, q, softmax_scale: float, *, out=None, lse=None,
               return_lse: bool = False, stream=None):
        """Absorbed causal attention of the step's queries ``q`` [tokens, heads,
        rank + rope] (the cache's type) over the cache, which holds the step's
        own rows.  Returns ``out`` [tokens, heads, rank] (also taken as an
        argument), with ``return_lse`` also the fp32 [tokens, heads] log-sum-exp
        of the scores.  Rows of torch tensors that are not 16-byte aligned are
        copied on the way."""
        batch._ready_for(self)
        d = batch._desc
        _latent_batch(batch)
        q, row = _aligned(q, "q", (d.tokens, d.heads, self.rank + self.rope), self.dtype, stream)
        _same_device(q, "q", self.device)
        out, to, result = _output(q, out, (d.tokens, d.heads, self.rank), self.dtype, self.device,
                                  stream)
        lse, lp = _statistics(q, lse, return_lse, (d.tokens, d.heads), self.device, stream)
        key = ("latent", self.rank, self.rope)
        need = batch._scratch.get(key)
        if need is None:
            got = u64()
            _lib.check(_call(self._lib.grm_hip_latent_attend_bytes, q, self.device, self._ref,
                             batch._ref, ctypes.byref(got)), "latent scratch size")
            need = batch._scratch[key] = got.value
        on = batch._on(q, stream)
        rc = _call(self._lib.grm_hip_latent_attend, q, self.device, self._ref, batch._ref,
                   batch._latent_at, batch._latent_bytes, *row, *to, lp, softmax_scale,
                   batch._scratch_on(q, need, on, stream) if need else None, need, on)
        if rc:
            _lib.check(rc, "latent attend")
        _written(out, result, on)
        return (out, lse) if return_lse else out

    def _ranges(self, block_table, starts, cu_rows, rows):
        n = int(starts.shape[0])
        table = _dense(block_table, "block_table", "i32", (n, block_table.shape[1]))
        sp = _dense(starts, "starts", "i32", (n,))
        cp = _dense(cu_rows, "cu_rows", "i32", (n + 1,))
        for a, what in ((block_table, "block_table"), (starts, "starts"), (cu_rows, "cu_rows")):
            _same_device(a, what, self.device)
        if not 0 <= int(rows) < 1 << 31:
            raise ValueError(f"rows must be 0 or more and fit 32 bits, got {rows}")
        return table, int(block_table.shape[1]), n, sp, cp, int(rows)

    def read(self, block_table, starts, cu_rows, rows: int, *, dtype=None, stream=None):
        """Dense rows [rows, rank + rope] of positions ``starts[r]`` onward of
        every request, ``cu_rows[r + 1] - cu_rows[r]`` of them; ``rows`` is
        ``cu_rows[-1]``.  In the cache's type unless told.  A deposit harvests a
        turn with it."""
        name = self.dtype if dtype is None else _name_of(dtype)
        if name not in ("f32", "bf16", "f16"):
            raise ValueError("rows are read as f32, bf16 or f16")
        at = self._ranges(block_table, starts, cu_rows, rows)
        out = _empty(starts, (at[5], self.rank + self.rope), name, stream)
        rc = _call(self._lib.grm_hip_latent_read, starts, self.device, self._ref, *at,
                   _lib.DTYPE_CODES[name], out.data_ptr(), _stream(starts, stream))
        if rc:
            _lib.check(rc, "latent read")
        return out

    def expand(self, weight, key_dim: int, block_table, starts, cu_rows, rows: int, *,
               stream=None):
        """A head's own keys and values, dense: (k [rows, heads, key_dim + rope],
        v [rows, heads, dim - key_dim]) of the positions that ``read`` would give,
        for ``weight`` [heads, dim, rank] of the cache's type, contiguous: its
        first ``key_dim`` rows make a head's keys (before the turned part), the
        others its values.  What prompts attend over with ``attend_rows``."""
        if len(weight.shape) != 3:
            raise ValueError("weight must be [heads, key_dim + value_dim, rank]")
        heads, dim = int(weight.shape[0]), int(weight.shape[1])
        key_dim = int(key_dim)
        if not 0 < key_dim < dim:
            raise ValueError(f"key_dim {key_dim} of {dim} rows a head")
        _no_gradient(weight, "weight")
        wp = _dense(weight, "weight", self.dtype, (heads, dim, self.rank))
        _same_device(weight, "weight", self.device)
        at = self._ranges(block_table, starts, cu_rows, rows)
        k = _empty(starts, (at[5], heads, key_dim + self.rope), self.dtype, stream)
        v = _empty(starts, (at[5], heads, dim - key_dim), self.dtype, stream)
        rc = _call(self._lib.grm_hip_latent_expand, starts, self.device, self._ref, wp, heads,
                   key_dim, dim - key_dim, *at, k.data_ptr(), v.data_ptr(), _stream(starts, stream))
        if rc:
            _lib.check(rc, "latent expand")
        return k, v


def attend_rows(batch: KvBatch, q, k, v, cu_rows, *, starts=None,
                softmax_scale: float | None = None, out=None, lse=None, return_lse: bool = False,
                stream=None):
    """Causal attention of a latent batch's queries ``q`` [tokens, heads, dk]
    over dense rows ``k`` [rows, heads, dk] and ``v`` [rows, heads, dv] (bf16 or
    f16, of one type), as ``LatentCache.expand`` makes them: request r's are
    ``cu_rows[r]`` to ``cu_rows[r + 1] - 1``, the first of them its position
    ``starts[r]`` (0 unless told).  Returns ``out`` [tokens, heads, dv] (also taken
    as an argument), with ``return_lse`` also the fp32 [tokens, heads]
    log-sum-exp, by which results over parts of the rows can be joined."""
    _latent_batch(batch)
    if not batch._planned:
        raise ValueError("the batch has no plan yet: call plan() first")
    d = batch._desc
    if len(k.shape) != 3 or len(v.shape) != 3:
        raise ValueError("k and v must be [rows, heads, dim]")
    rows, dk, dv = int(k.shape[0]), int(k.shape[2]), int(v.shape[2])
    name = _type(q, "q")
    if name not in ("bf16", "f16"):
        raise ValueError(f"q must be bf16 or f16, got {q.dtype}")
    q, at_q = _aligned(q, "q", (d.tokens, d.heads, dk), name, stream)
    k, at_k = _aligned(k, "k", (rows, d.heads, dk), name, stream)
    v, at_v = _aligned(v, "v", (rows, d.heads, dv), name, stream)
    cu = _dense(cu_rows, "cu_rows", "i32", (d.requests + 1,))
    sp = None if starts is None else _dense(starts, "starts", "i32", (d.requests,))
    for a, what in ((q, "q"), (k, "k"), (v, "v"), (cu_rows, "cu_rows"), (starts, "starts")):
        if a is not None:
            _same_device(a, what, batch.device)
    out, to, result = _output(q, out, (d.tokens, d.heads, dv), name, batch.device, stream)
    lse, lp = _statistics(q, lse, return_lse, (d.tokens, d.heads), batch.device, stream)
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(dk)
    key = ("rows", dk, dv)
    need = batch._scratch.get(key)
    if need is None:
        got = u64()
        _lib.check(_call(batch._lib.grm_hip_rows_attend_bytes, q, batch.device, batch._ref, dk, dv,
                         ctypes.byref(got)), "rows scratch size")
        need = batch._scratch[key] = got.value
    on = batch._on(q, stream)
    rc = _call(batch._lib.grm_hip_rows_attend, q, batch.device, batch._ref, batch._latent_at,
               batch._latent_bytes, _lib.DTYPE_CODES[name], dk, dv, *at_q, *at_k, *at_v, rows, cu,
               sp, *to, lp, softmax_scale,
               batch._scratch_on(q, need, on, stream) if need else None, need, on)
    if rc:
        _lib.check(rc, "rows attend")
    _written(out, result, on)
    return (out, lse) if return_lse else out


__all__ = ["LatentCache", "attend_rows"]
