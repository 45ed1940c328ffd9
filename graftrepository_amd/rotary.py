"""Rotary positions: pairs of channels turned by an angle that grows with the
position.

A graft's keys are stored as they were harvested and mounted at other
positions; ``Rotary`` says how a model turns keys and queries to theirs::

    rotary = Rotary(128)                            # halves as pairs, base 10000
    q = rotary.apply(q, batch.positions)            # queries of a step
    cache.append(batch, k, v, rotary=rotary)        # keys, on their way into a cache
    raw = rotary.apply(k, positions, inverse=True)  # a harvest, turned back

Pair i of ``dim`` channels turns by ``position * f_i``, f_i = base^(-2 i /
dim), and grows by ``magnitude``.  Pairs are channels (i, i + dim/2), or (2 i,
2 i + 1) with ``layout="interleaved"``.  ``scaling`` reaches positions past
the ``trained`` ones:

* ``"linear"``: f / factor;
* ``"base"``: base * factor^(dim / (dim - 2));
* ``"yarn"``: f that turn more than ``fast`` times in ``trained`` positions
  stay, f that turn less than ``slow`` times become f / factor, with a ramp over
  the pairs between; magnitude 0.1 ln(factor) + 1 unless given;
* ``"smooth"``: the same ends, with a ramp over the number of turns;
* ``"factors"``: f_i / factors[i].

Angles are made in fp64 on the device, so there is no table and no last
position.  The laws are those of ``include/grm_hip_router.h``.
"""

from __future__ import annotations

import ctypes
import math

from . import _lib
from .kv_cache import (_call, _dense, _empty, _one_device, _rows, _same_device, _size, _stream)


class _RotaryDesc(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_double * 128), ("magnitude", ctypes.c_float),
                ("dim", ctypes.c_int32), ("layout", ctypes.c_int32), ("inverse", ctypes.c_int32)]


def _frequencies(dim, base, scaling, factor, trained, fast, slow, factors):
    pairs = range(dim // 2)
    if scaling == "base":
        if dim == 2:
            raise ValueError("scaling 'base' needs dim of 4 or more")
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in pairs]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "yarn":
        def pair(turns):  # the pair (a real number) that turns so often
            return dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair(fast)), 0)
        high = min(math.ceil(pair(slow)), dim - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in pairs]
        return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)]
    if scaling == "smooth":
        stay = [(x * trained / (2 * math.pi) - slow) / (fast - slow) for x in f]
        stay = [min(max(s, 0.0), 1.0) for s in stay]
        return [x / factor * (1 - s) + x * s for x, s in zip(f, stay)]
    if scaling == "factors":
        if factors is None or len(factors) != dim // 2:
            raise ValueError(f"scaling 'factors' needs dim / 2 = {dim // 2} of them")
        return [x / float(g) for x, g in zip(f, factors)]
    return f


class Rotary:
    """How ``dim`` channels of a head are turned; see the module."""

    def __init__(self, dim: int, *, base: float = 10000.0, layout: str = "half",
                 scaling: str | None = None, factor: float = 1.0, trained: int = 4096,
                 fast: float = 32.0, slow: float = 1.0, factors=None,
                 magnitude: float | None = None):
        dim = int(dim)
        if dim % 2 or not 2 <= dim <= 256:
            raise ValueError(f"dim must be even, 2 to 256, got {dim}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if scaling not in (None, "linear", "base", "yarn", "smooth", "factors"):
            raise ValueError(f"unknown scaling {scaling!r}")
        if not (base > 1 and math.isfinite(base)):
            raise ValueError(f"base must be finite and above 1, got {base}")
        if not (factor > 0 and math.isfinite(factor)):
            raise ValueError(f"factor must be positive and finite, got {factor}")
        if not (0 < trained < math.inf and 0 < slow < fast < math.inf):
            raise ValueError("trained must be positive, 0 < slow < fast, and all finite")
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1 else 1.0
        if not 1e-30 < magnitude < 1e30:
            raise ValueError(f"magnitude must be positive and finite, got {magnitude}")
        self.dim, self.layout, self.magnitude = dim, layout, magnitude
        try:
            self.frequencies = _frequencies(dim, float(base), scaling, float(factor), trained,
                                            fast, slow, factors)
        except ArithmeticError as e:  # a factor of 0, a base past fp64's range
            raise ValueError(f"no frequencies of these arguments: {e}") from None
        if not all(math.isfinite(f) and abs(f) <= 2 * math.pi for f in self.frequencies):
            raise ValueError("a frequency past one turn a position")
        self._desc = {}
        for inverse in (False, True):
            d = _RotaryDesc()
            d.turns[:dim // 2] = [f / (2 * math.pi) for f in self.frequencies]
            d.magnitude, d.dim, d.layout = magnitude, dim, int(layout == "interleaved")
            d.inverse = int(inverse)
            self._desc[inverse] = d
        self._refs = tuple(ctypes.byref(d) for d in self._desc.values())
        self._ref = self._refs[0]
        self._rotate = None  # the library's entry, from the first call on

    def apply(self, x, positions, *, start: int = 0, out=None, inverse: bool = False, stream=None):
        """``x`` [tokens, heads, head_dim] (f32, bf16 or f16; any row and head
        strides) with channels [start, start + dim) of every head turned to
        ``positions`` int32 [tokens]; the others are copied.  ``out`` (x's type
        and shape) may be ``x``.  ``inverse`` undoes it.  Rows whose position is
        below 0 (a batch's rows past its last token) are not written."""
        shape = tuple(x.shape)
        if len(shape) != 3:
            raise ValueError(f"x must be [tokens, heads, head_dim], got {shape}")
        start = _size(start, "start")
        if start < 0 or start + self.dim > shape[2]:
            raise ValueError(f"channels {start} to {start + self.dim} of heads of {shape[2]}")
        xp, name, xt, xh = _rows(x, "x", shape, "rotation")
        pos = _dense(positions, "positions", "i32", (shape[0],))
        device = x.get_device()
        _same_device(positions, "positions", device)
        if out is None:
            out = _empty(x, shape, name, stream)
            op, ot, oh = out.data_ptr(), shape[1] * shape[2], shape[2]
        elif out is x:
            op, ot, oh = xp, xt, xh
        else:
            op, oname, ot, oh = _rows(out, "out", shape, "rotation")
            if oname != name:
                raise ValueError("out must have x's type")
            _one_device(x=x, out=out)
        if shape[0] and shape[1]:
            if self._rotate is None:
                self._rotate = _lib.load().grm_hip_rotate
            rc = _call(self._rotate, x, device, self._refs[bool(inverse)], xp,
                       _lib.DTYPE_CODES[name], xt, xh, op, ot, oh, pos, shape[0], shape[1],
                       shape[2], start, _stream(x, stream))
            if rc:
                _lib.check(rc, "rotate")
        return out


__all__ = ["Rotary"]
