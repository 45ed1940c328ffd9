"""A paged key/value cache held in 8 bits, and attention over it.

Routed grafts end up in the model's cache (the reference mounts them by
surgery on a dense fp16 cache, core/graft_arena.py:2408-2622, and leaves the
attention to its external engine).  ``KvCache`` holds keys and values as int8
codes with one fp32 scale per (block of tokens, kv head); ``KvBatch`` is one
step's ragged batch over it::

    batch = KvBatch(ctx_lens, new_lens, block_table, 64, tokens=T, max_new=n,
                    heads=32, kv_heads=8, free_list=free, free_head=head)
    batch.plan()                          # once per step
    cache.append(batch, k, v)             # per layer
    out = cache.attend(batch, q)          # per layer
    k, v = cache.read(table, starts, cu_rows, rows)   # dense, to harvest

Arrays are device memory: torch tensors, or ``payload.DeviceArray`` (there
bf16 is uint16 bit patterns, as everywhere in this package; a layer of an
unpacked node goes to ``append`` as ``node["k"].rows(layer)``).  Shapes, laws
and layouts are those of ``include/grm_hip_router.h``.  All arrays of a batch,
its caches and its calls are on one GPU, which need not be the current one for
torch tensors; DeviceArrays are used with theirs current.  Calls are ordered on
``stream`` (a HIP stream handle; by default torch's current stream for torch
tensors, else the default stream) and return before the work has run; they
can be captured into a HIP graph.  There is no backward pass: values that
require a gradient are refused where gradients are recorded.  Bad arguments raise ``ValueError`` here or
``RuntimeError`` (code -1) from the library, with nothing launched.
"""

from __future__ import annotations

import ctypes
import math
import sys

import numpy as np

from . import _lib
from .payload import DeviceArray, DeviceRows, current_device

i32, u64, vp = ctypes.c_int32, ctypes.c_uint64, ctypes.c_void_p


class _CacheDesc(ctypes.Structure):
    _fields_ = [("k_codes", vp), ("v_codes", vp), ("k_scales", vp), ("v_scales", vp),
                ("blocks", u64), ("block_tokens", i32), ("kv_heads", i32), ("head_dim", i32),
                ("reserved", i32)]


class _BatchDesc(ctypes.Structure):
    _fields_ = [("ctx_lens", vp), ("new_lens", vp), ("block_table", vp), ("free_list", vp),
                ("free_head", vp), ("free_head_out", vp), ("cu_new", vp), ("slot_map", vp),
                ("positions", vp), ("work", vp), ("work_bytes", u64), ("requests", i32),
                ("table_width", i32), ("tokens", i32), ("max_new", i32), ("block_tokens", i32),
                ("heads", i32), ("kv_heads", i32), ("window", i32), ("free_count", u64)]


_NUMPY = {"f32": np.float32, "bf16": np.uint16, "f16": np.float16, "i8": np.int8,
          "i32": np.int32, "i64": np.int64, "u8": np.uint8}
_NAMES = {np.dtype(v): k for k, v in _NUMPY.items()}
_TORCH: dict[str, object] = {}
_FLOATS: dict[object, str] = {}   # torch's floating types, once torch is there


def _torch_names() -> dict[str, object]:
    if not _TORCH:
        t = sys.modules["torch"]
        pairs = {"f32": t.float32, "bf16": t.bfloat16, "f16": t.float16, "i8": t.int8,
                 "i32": t.int32, "i64": t.int64, "u8": t.uint8}
        _NAMES.update({v: k for k, v in pairs.items()})
        _FLOATS.update({pairs[k]: k for k in ("f32", "bf16", "f16")})
        _TORCH.update(pairs)
    return _TORCH


def _size(n, what: str) -> int:
    """A size for a field of 32 bits, which ctypes would cut to them."""
    n = int(n)
    if not -(1 << 31) <= n < 1 << 31:
        raise ValueError(f"{what} must fit 32 bits, got {n}")
    return n


def _is_torch(a) -> bool:
    t = sys.modules.get("torch")
    return t is not None and isinstance(a, t.Tensor)


def _name_of(dtype) -> str:
    """'bf16' and the like of a name, a numpy or a torch type."""
    if isinstance(dtype, str) and dtype in _NUMPY:
        return dtype
    if "torch" in sys.modules:
        _torch_names()
    try:
        return _NAMES[dtype] if dtype in _NAMES else _NAMES[np.dtype(dtype)]
    except (KeyError, TypeError):
        raise ValueError(f"unsupported type {dtype!r}") from None


def _type(a, what: str) -> str:
    if _is_torch(a):
        _torch_names()
        if not a.is_cuda:
            raise ValueError(f"{what} must be on the GPU")
    elif not isinstance(a, (DeviceArray, DeviceRows)):
        raise ValueError(f"{what} must be a torch tensor on the GPU or a DeviceArray")
    name = _NAMES.get(a.dtype)
    if name is None:
        raise ValueError(f"{what}: unsupported type {a.dtype}")
    return name


def _dense(a, what: str, dtype: str, shape) -> int:
    """Address of a contiguous array of this type and shape (None: any)."""
    if _TORCH and getattr(a, "dtype", None) is _TORCH[dtype] and a.is_cuda and \
            a.shape == shape and a.is_contiguous():
        return a.data_ptr()  # the usual call, on its short way
    if _type(a, what) != dtype:
        raise ValueError(f"{what} must be {dtype}, got {a.dtype}")
    got = tuple(a.shape)
    if len(got) != len(shape) or any(w is not None and g != w for g, w in zip(got, shape)):
        raise ValueError(f"{what} must have shape {shape}, got {got}")
    if not a.is_contiguous() if _is_torch(a) else isinstance(a, DeviceRows):
        raise ValueError(f"{what} must be contiguous")
    return a.data_ptr()


def _strides(a) -> tuple[int, ...]:
    if _is_torch(a):
        return a.stride()
    if isinstance(a, DeviceRows):
        return a.strides
    out, step = [], 1
    for d in reversed(a.shape):
        out.append(step)
        step *= d
    return tuple(reversed(out))


def _rows(a, what: str, shape) -> tuple[int, str, int, int]:
    """(address, type, row stride, head stride) of [rows, heads, dim] values
    whose last axis is contiguous."""
    if getattr(a, "requires_grad", False) and sys.modules["torch"].is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and the cache has no backward pass: "
                         "detach it, or call under torch.no_grad()")
    if _FLOATS and _FLOATS.get(getattr(a, "dtype", None)) and a.is_cuda and a.shape == shape:
        st = a.stride()
        if st[2] == 1:  # the usual call, on its short way
            return a.data_ptr(), _FLOATS[a.dtype], st[0], st[1]
    name = _type(a, what)
    if name not in ("f32", "bf16", "f16"):
        raise ValueError(f"{what} must be f32, bf16 or f16, got {a.dtype}")
    if tuple(a.shape) != shape:
        raise ValueError(f"{what} must have shape {shape}, got {tuple(a.shape)}")
    st = _strides(a)
    if st[2] != 1 and shape[2] > 1 and a.data_ptr():
        raise ValueError(f"{what}: the last axis must be contiguous")
    return a.data_ptr(), name, st[0], st[1]


def _off(row) -> bool:
    """Whether such rows (address, type, strides) are not 16-byte aligned."""
    ptr, name, token, head = row
    return bool(ptr & 15 or (token | head) & (3 if name == "f32" else 7))


def _copied(a, stream):
    """A torch tensor's values, contiguous, made on the stream of the call."""
    t = sys.modules["torch"]
    with t.cuda.stream(_torch_stream(a, _stream(a, stream))):
        return a.clone(memory_format=t.contiguous_format)


def _empty(like, shape, dtype: str, stream=None):
    """Memory beside ``like``.  Torch's belongs to the stream that the call
    uses, since that is where its last use is when it is freed."""
    if not _is_torch(like):
        return DeviceArray(shape, _NUMPY[dtype])
    t = sys.modules["torch"]
    if stream is None:
        return t.empty(shape, dtype=_torch_names()[dtype], device=like.device)
    with t.cuda.stream(_torch_stream(like, _stream(like, stream))):
        return t.empty(shape, dtype=_torch_names()[dtype], device=like.device)


def _one_device(**arrays) -> int:
    """The device that all of these are on."""
    on = {what: a.get_device() for what, a in arrays.items() if a is not None}
    if len(set(on.values())) != 1:
        raise ValueError(f"arrays are on more than one GPU: {on}")
    return next(iter(on.values()))


def _same_device(a, what: str, device: int) -> None:
    if a.get_device() != device:
        raise ValueError(f"{what} is on GPU {a.get_device()}, the batch or cache on GPU {device}")


def _find_torch_device() -> int:
    global _torch_device
    t = sys.modules["torch"]
    _torch_device = getattr(t._C, "_cuda_getDevice", None) or t.cuda.current_device
    return _torch_device()


_torch_device = _find_torch_device  # torch's current device


def _call(fn, like, device: int, *args) -> int:
    """fn(*args) with the arrays' device current, which the library launches on."""
    if isinstance(like, (DeviceArray, DeviceRows)):
        here = current_device()
        if here != device:
            raise ValueError(f"the arrays are on GPU {device}, the current device is GPU {here}")
    elif _torch_device() != device:
        with sys.modules["torch"].cuda.device(device):
            return fn(*args)
    return fn(*args)


def _torch_stream(like, on: int):
    """The stream of this handle, on the tensor's device."""
    t = sys.modules["torch"]
    return t.cuda.ExternalStream(on, like.device) if on else t.cuda.default_stream(like.device)


_raw_stream = None  # torch's current stream of a device as a handle


def _stream(a, stream) -> int:
    global _raw_stream
    if stream is not None:
        if not isinstance(stream, int) and getattr(stream, "device_index", a.get_device()) != a.get_device():
            raise ValueError(f"a stream of GPU {stream.device_index} for arrays on GPU "
                             f"{a.get_device()}")
        return int(getattr(stream, "cuda_stream", stream))
    if isinstance(a, (DeviceArray, DeviceRows)):
        return 0
    if _raw_stream is None:
        t = sys.modules["torch"]
        _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: t.cuda.current_stream(i).cuda_stream)
    return _raw_stream(a.get_device())


class KvBatch:
    """One step's ragged batch: request r holds ``ctx_lens[r]`` tokens and
    brings ``new_lens[r]``; its tokens are rows ``cu_new[r]`` onward.

    ``block_table`` int32 [requests, width]: physical block of each of a
    request's blocks.  With ``free_list`` (int32) and ``free_head`` (int32
    [1], entries used so far), ``plan`` takes the blocks that are missing
    from the list, enters them in the table and leaves the new head in
    ``free_head_out``; ``advance`` makes that the next plan's head.  Without a
    list the table is taken as it is.

    ``tokens`` is the number of rows of the step's arrays (at least the sum
    of ``new_lens``) and ``max_new`` a bound on its entries: both fix grids
    and buffers, so a batch object serves every step within them, with
    ``ctx_lens``, ``new_lens`` and the table updated in place.  ``window``
    limits a token to its last ``window`` tokens; layers with another window
    take a second batch over the same arrays.

    Calls with one batch follow each other: on one stream, or ordered by the
    caller.  Work that runs at the same time on several streams, replays of
    captured graphs included, takes a batch each, and a graph's batch stays
    as long as the graph.
    """

    def __init__(self, ctx_lens, new_lens, block_table, block_tokens: int, *, tokens: int,
                 max_new: int, heads: int, kv_heads: int, window: int = 0, free_list=None,
                 free_head=None):
        self._lib = _lib.load()
        n = int(ctx_lens.shape[0])
        d = self._desc = _BatchDesc()
        d.ctx_lens = _dense(ctx_lens, "ctx_lens", "i32", (n,))
        d.new_lens = _dense(new_lens, "new_lens", "i32", (n,))
        d.block_table = _dense(block_table, "block_table", "i32", (n, None))
        d.requests, d.table_width = n, int(block_table.shape[1])
        for what, size in (("tokens", tokens), ("max_new", max_new), ("window", window),
                           ("block_tokens", block_tokens), ("heads", heads),
                           ("kv_heads", kv_heads)):
            setattr(d, what, _size(size, what))
        self.device = _one_device(ctx_lens=ctx_lens, new_lens=new_lens, block_table=block_table,
                                  free_list=free_list, free_head=free_head)
        need = u64()
        _lib.check(_call(self._lib.grm_hip_kv_work_bytes, ctx_lens, self.device, ctypes.byref(d),
                         ctypes.byref(need)), "kv work size")
        self.ctx_lens, self.new_lens, self.block_table = ctx_lens, new_lens, block_table
        self.cu_new = _empty(ctx_lens, (n + 1,), "i32")
        self.slot_map = _empty(ctx_lens, (d.tokens,), "i64")
        self.positions = _empty(ctx_lens, (d.tokens,), "i32")
        self._work = _empty(ctx_lens, (need.value,), "u8")
        d.cu_new, d.slot_map = self.cu_new.data_ptr(), self.slot_map.data_ptr()
        d.positions, d.work = self.positions.data_ptr(), self._work.data_ptr()
        d.work_bytes = need.value
        self.free_list = self.free_head = self.free_head_out = self._made_head = None
        if free_list is not None:
            if free_head is None:
                raise ValueError("a free list needs free_head")
            d.free_list = _dense(free_list, "free_list", "i32", (None,))
            d.free_count = int(free_list.shape[0])
            d.free_head = _dense(free_head, "free_head", "i32", (1,))
            self.free_list, self.free_head = free_list, free_head
            self.free_head_out = self._made_head = _empty(ctx_lens, (1,), "i32")
            d.free_head_out = self.free_head_out.data_ptr()
        self._ref = ctypes.byref(d)
        self._scratch: dict[int, int] = {}
        self._held: dict[int, list] = {}
        self._streams = {_stream(ctx_lens, None)}
        self._planned = False  # once
        self._taken = False    # since the free list last went on

    def plan(self, stream=None) -> "KvBatch":
        """Fill ``cu_new``, ``slot_map``, ``positions``, the table's new
        entries and the schedule from the lengths as they are now."""
        rc = _call(self._lib.grm_hip_kv_plan, self.ctx_lens, self.device, self._ref,
                   self._on(self.ctx_lens, stream))
        if rc:
            _lib.check(rc, "kv plan")
        self._planned = self._taken = True
        return self

    def _scratch_on(self, like, need: int, on: int, stream) -> int:
        """Scratch of a call, the largest of its stream: calls on one stream
        follow each other and may share it.  What a call was given stays for
        the batch's life, since a captured graph goes on writing to it."""
        held = self._held.setdefault(on, [])
        if not held or held[-1].nbytes < need:
            held.append(_empty(like, (need,), "u8", stream))
        return held[-1].data_ptr()

    def _on(self, like, stream) -> int:
        """The stream a call runs on.  What this object made is torch's to hand
        out again once it is dropped, but not before that stream is through
        with it."""
        on = _stream(like, stream)
        if on not in self._streams:
            self._streams.add(on)
            if _is_torch(self._work):
                s = _torch_stream(self._work, on)
                for a in (self.cu_new, self.slot_map, self.positions, self._work,
                          self._made_head):
                    if a is not None:
                        a.record_stream(s)
        return on

    def _ready_for(self, cache):
        if cache.device != self.device:
            raise ValueError(f"the cache is on GPU {cache.device}, the batch on GPU {self.device}")
        if not self._planned:
            raise ValueError("the batch has no plan yet: call plan() first")

    def advance(self) -> None:
        """The next plan goes on in the free list where the last one ended."""
        if self.free_list is None:
            raise ValueError("the batch has no free list")
        if not self._taken:
            raise ValueError("no plan since the last advance: the list would go back to where "
                             "that began, and hand its blocks out again")
        self._taken = False
        d = self._desc
        self.free_head, self.free_head_out = self.free_head_out, self.free_head
        d.free_head, d.free_head_out = d.free_head_out, d.free_head


class KvCache:
    """The cache of one layer, over the caller's arrays: int8 ``k_codes``
    [blocks, kv_heads, block_tokens, head_dim] and ``v_codes`` [blocks,
    kv_heads, head_dim, block_tokens] (transposed in its block), fp32
    ``k_scales`` and ``v_scales`` [blocks, kv_heads], 0, positive or NaN.
    ``KvCache.empty`` allocates them."""

    def __init__(self, k_codes, v_codes, k_scales, v_scales):
        self._lib = _lib.load()
        if len(k_codes.shape) != 4:
            raise ValueError("k_codes must be [blocks, kv_heads, block_tokens, head_dim]")
        blocks, kv, bs, hd = (int(s) for s in k_codes.shape)
        d = self._desc = _CacheDesc()
        d.k_codes = _dense(k_codes, "k_codes", "i8", (blocks, kv, bs, hd))
        d.v_codes = _dense(v_codes, "v_codes", "i8", (blocks, kv, hd, bs))
        d.k_scales = _dense(k_scales, "k_scales", "f32", (blocks, kv))
        d.v_scales = _dense(v_scales, "v_scales", "f32", (blocks, kv))
        self.device = _one_device(k_codes=k_codes, v_codes=v_codes, k_scales=k_scales,
                                  v_scales=v_scales)
        d.blocks, d.block_tokens, d.kv_heads, d.head_dim = blocks, bs, kv, hd
        if bs not in (16, 32, 64, 128):
            raise ValueError("block_tokens must be 16, 32, 64 or 128")
        if hd % 16 or not 0 < hd <= 256:
            raise ValueError("head_dim must be a multiple of 16, at most 256")
        self.k_codes, self.v_codes = k_codes, v_codes
        self.k_scales, self.v_scales = k_scales, v_scales
        self.blocks, self.block_tokens, self.kv_heads, self.head_dim = blocks, bs, kv, hd
        self._ref = ctypes.byref(d)

    @classmethod
    def empty(cls, blocks: int, block_tokens: int, kv_heads: int, head_dim: int) -> "KvCache":
        """A cache in memory of its own (DeviceArrays), contents undefined:
        every block is written before it is read."""
        k = DeviceArray((blocks, kv_heads, block_tokens, head_dim), np.int8)
        v = DeviceArray((blocks, kv_heads, head_dim, block_tokens), np.int8)
        ks = DeviceArray((blocks, kv_heads), np.float32)
        return cls(k, v, ks, DeviceArray((blocks, kv_heads), np.float32))

    def append(self, batch: KvBatch, k, v, stream=None) -> None:
        """Quantise the step's ``k`` and ``v`` [tokens, kv_heads, head_dim]
        (f32, bf16 or f16; any row and head strides) into their blocks."""
        batch._ready_for(self)
        shape = (batch._desc.tokens, self.kv_heads, self.head_dim)
        kp, name, kt, kh = _rows(k, "k", shape)
        vptr, vname, vt, vh = _rows(v, "v", shape)
        if vname != name:
            raise ValueError("k and v must have one type")
        _same_device(k, "k", self.device)
        _same_device(v, "v", self.device)
        rc = _call(self._lib.grm_hip_kv_append, k, self.device, self._ref, batch._ref, kp, vptr,
                   _lib.DTYPE_CODES[name], kt, kh, vt, vh, batch._on(k, stream))
        if rc:
            _lib.check(rc, "kv append")

    def attend(self, batch: KvBatch, q, softmax_scale: float | None = None, *, out=None,
               lse=None, return_lse: bool = False, stream=None):
        """Causal attention of the step's queries ``q`` [tokens, heads,
        head_dim] over the cache, which holds the step's own tokens.  Returns
        ``out`` (q's type; also taken as an argument), with ``return_lse``
        also the fp32 [tokens, heads] log-sum-exp of the scores.  Rows of torch
        tensors that are not 16-byte aligned are copied on the way."""
        batch._ready_for(self)
        d = batch._desc
        shape = (d.tokens, d.heads, self.head_dim)
        row = _rows(q, "q", shape)
        if _off(row) and _is_torch(q):
            q = _copied(q, stream)
            row = _rows(q, "q", shape)
        qp, name, qt, qh = row
        if q.get_device() != self.device:
            _same_device(q, "q", self.device)
        result = None   # what an output of other rows is copied from
        if out is None:
            out = _empty(q, shape, name, stream)
            op, ot, oh = out.data_ptr(), shape[1] * shape[2], shape[2]
        else:
            row = _rows(out, "out", shape)
            if _off(row) and _is_torch(out):
                result = _copied(out, stream)   # rows that are not written stay
                row = _rows(result, "out", shape)
            op, oname, ot, oh = row
            if oname != name:
                raise ValueError("out must have q's type")
            _same_device(out, "out", self.device)
        if lse is None and return_lse:
            lse = _empty(q, shape[:2], "f32", stream)
            lp = lse.data_ptr()
        else:
            lp = _dense(lse, "lse", "f32", shape[:2]) if lse is not None else None
            if lse is not None:
                _same_device(lse, "lse", self.device)
        need = batch._scratch.get(self.head_dim)
        if need is None:
            got = u64()
            _lib.check(_call(self._lib.grm_hip_kv_attend_bytes, q, self.device, self._ref,
                             batch._ref, ctypes.byref(got)), "kv scratch size")
            need = batch._scratch[self.head_dim] = got.value
        if softmax_scale is None:
            softmax_scale = 1.0 / math.sqrt(self.head_dim)
        on = batch._on(q, stream)
        rc = _call(
            self._lib.grm_hip_kv_attend, q, self.device, self._ref, batch._ref, qp,
            _lib.DTYPE_CODES[name], qt, qh, op, ot, oh, lp, softmax_scale,
            batch._scratch_on(q, need, on, stream) if need else None, need, on)
        if rc:
            _lib.check(rc, "kv attend")
        if result is not None:
            with sys.modules["torch"].cuda.stream(_torch_stream(out, on)):
                out.copy_(result)
        return (out, lse) if return_lse else out

    def read(self, block_table, starts, cu_rows, rows: int, *, dtype="f16", stream=None):
        """Dense (k, v) [rows, kv_heads, head_dim] of positions ``starts[r]``
        onward of every request, ``cu_rows[r + 1] - cu_rows[r]`` of them;
        ``rows`` is ``cu_rows[-1]``.  A deposit harvests a turn with it."""
        name = _name_of(dtype)
        if name not in ("f32", "bf16", "f16"):
            raise ValueError("values are read as f32, bf16 or f16")
        n = int(starts.shape[0])
        table = _dense(block_table, "block_table", "i32", (n, block_table.shape[1]))
        sp = _dense(starts, "starts", "i32", (n,))
        cp = _dense(cu_rows, "cu_rows", "i32", (n + 1,))
        for a, what in ((block_table, "block_table"), (starts, "starts"), (cu_rows, "cu_rows")):
            _same_device(a, what, self.device)
        if not 0 <= int(rows) < 1 << 31:
            raise ValueError(f"rows must be 0 or more and fit 32 bits, got {rows}")
        shape = (int(rows), self.kv_heads, self.head_dim)
        k, v = _empty(starts, shape, name, stream), _empty(starts, shape, name, stream)
        rc = _call(
            self._lib.grm_hip_kv_read, starts, self.device, self._ref, table,
            int(block_table.shape[1]), n, sp, cp, shape[0], _lib.DTYPE_CODES[name], k.data_ptr(),
            v.data_ptr(), _stream(starts, stream))
        if rc:
            _lib.check(rc, "kv read")
        return k, v


__all__ = ["KvBatch", "KvCache"]
