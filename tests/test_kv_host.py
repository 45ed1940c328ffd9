"""What the key/value cache's Python side keeps and checks on the host, with a
library and arrays that only write down what they are asked (CPU only)."""

import ctypes
import gc
import weakref

import numpy as np
import pytest

import graftrepository_amd as g
from graftrepository_amd import kv_cache as kc
from tests.test_kv_cache import fake


class Lib:
    """The library's key/value entries: sizes by head_dim, calls written down."""

    def __init__(self):
        self.calls = []

    def grm_hip_kv_work_bytes(self, batch, out):
        out._obj.value = 640
        return 0

    def grm_hip_kv_attend_bytes(self, cache, batch, out):
        out._obj.value = 1000 * cache._obj.head_dim
        return 0

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    lib, places = Lib(), iter(range(1, 1 << 30))
    monkeypatch.setattr(kc._lib, "load", lambda: lib)

    def empty(like, shape, dtype, stream=None):
        a = fake(shape, kc._NUMPY[dtype])
        a.ptr = next(places) << 12
        lib.made.append(weakref.ref(a))
        return a
    lib.made = []
    monkeypatch.setattr(kc, "_empty", empty)
    return lib


def cache_of(hd, kv=2):
    return g.KvCache(fake((4, kv, 16, hd), np.int8), fake((4, kv, hd, 16), np.int8),
                     fake((4, kv), np.float32), fake((4, kv), np.float32))


def batch_of(tokens=3, **kw):
    kw = {**dict(tokens=tokens, max_new=1, heads=4, kv_heads=2), **kw}
    return g.KvBatch(fake((3,), np.int32), fake((3,), np.int32), fake((3, 4), np.int32), 16, **kw)


def test_scratch_that_was_handed_out_stays_as_long_as_its_batch(lib):
    """A captured graph holds the address of the scratch that its call was
    given: a later call that needs more must not free it."""
    b = batch_of().plan()
    given = []
    for hd in (64, 256, 128, 64):
        cache_of(hd).attend(b, fake((3, 4, hd), np.float32))
        args = lib.calls[-1][1]
        given.append((args[11], args[12]))
    gc.collect()
    there = {r().ptr: r().nbytes for r in lib.made if r() is not None}
    for ptr, need in given:
        assert there.get(ptr, 0) >= need
    assert len({p for p, _ in given[1:]}) == 1     # and what is large enough serves again


def test_a_refused_attend_leaves_no_size_behind(lib):
    """The scratch's size is kept by head_dim: one asked with a cache that does
    not fit the batch must not be."""
    b, sizes = batch_of().plan(), []

    def attend_bytes(cache, batch, out):
        if cache._obj.kv_heads != batch._obj.kv_heads:
            return -1
        out._obj.value = 4096
        sizes.append(1)
        return 0
    lib.grm_hip_kv_attend_bytes = attend_bytes
    with pytest.raises(RuntimeError):
        cache_of(64, kv=1).attend(b, fake((3, 4, 64), np.float32))
    cache_of(64).attend(b, fake((3, 4, 64), np.float32))
    assert sizes == [1] and lib.calls[-1][1][12] == 4096


@pytest.mark.parametrize("change", [dict(kv_heads=4), dict(block_tokens=32)])
def test_scratch_of_a_cache_that_does_not_fit_is_refused(change):
    real = g.load()
    from tests.test_kv_cache import batch_desc, cache_desc
    out = ctypes.c_uint64(7)
    assert real.grm_hip_kv_attend_bytes(ctypes.byref(cache_desc(**change)),
                                        ctypes.byref(batch_desc()), ctypes.byref(out)) == -1
    assert b"differ" in real.grm_hip_last_error() and out.value == 7


def test_a_batch_is_kept_for_the_streams_that_read_it(lib, monkeypatch):
    """The schedule and the other arrays that a batch made are recorded for every
    stream that a call names, beside the one that they were made on."""
    kept = []

    class Tensorlike:
        """An array that is torch's, as far as this side asks."""

        def __init__(self, shape, dtype):
            self.shape, self.dtype, self.is_cuda = tuple(shape), np.dtype(dtype), True
            self.nbytes = int(np.prod(shape)) * self.dtype.itemsize

        data_ptr = lambda self: 0x1000        # noqa: E731
        get_device = lambda self: 0           # noqa: E731
        is_contiguous = lambda self: True     # noqa: E731

        def stride(self):
            return tuple(np.cumprod((1, *self.shape[:0:-1]))[::-1].tolist())

        def record_stream(self, s):
            kept.append((id(self), s))

    monkeypatch.setattr(kc, "_is_torch", lambda a: isinstance(a, Tensorlike))
    monkeypatch.setattr(kc, "_torch_names", lambda: kc._TORCH)
    monkeypatch.setattr(kc, "_empty", lambda like, shape, dtype, stream=None: Tensorlike(
        shape, kc._NUMPY[dtype]))
    monkeypatch.setattr(kc, "_stream", lambda a, stream: 5 if stream is None else stream)
    monkeypatch.setattr(kc, "_torch_stream", lambda a, on: ("stream", on))
    T = Tensorlike
    b = g.KvBatch(T((3,), np.int32), T((3,), np.int32), T((3, 4), np.int32), 16, tokens=3,
                  max_new=1, heads=4, kv_heads=2, free_list=T((9,), np.int32),
                  free_head=T((1,), np.int32))
    mine = {id(a) for a in (b.cu_new, b.slot_map, b.positions, b._work, b.free_head_out)}
    c = g.KvCache(T((4, 2, 16, 64), np.int8), T((4, 2, 64, 16), np.int8), T((4, 2), np.float32),
                  T((4, 2), np.float32))
    b.plan()
    b.plan(stream=5)
    assert not kept                                # where they were made
    b.plan(stream=7)
    assert {i for i, _ in kept} == mine and {s for _, s in kept} == {("stream", 7)}
    c.append(b, T((3, 2, 64), np.float32), T((3, 2, 64), np.float32), stream=7)
    assert len(kept) == len(mine)                  # once is enough
    c.append(b, T((3, 2, 64), np.float32), T((3, 2, 64), np.float32), stream=8)
    assert kept[-1][1] == ("stream", 8)
    c.attend(b, T((3, 4, 64), np.float32), stream=0)
    assert {i for i, s in kept if s == ("stream", 0)} == mine
