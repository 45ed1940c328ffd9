"""What the key/value cache's Python side keeps and checks on the host, with a
library and arrays that only write down what they are asked (CPU only)."""

import contextlib
import ctypes
import gc
import sys
import types
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


class Tensorlike:
    """An array that is torch's, as far as this side asks."""

    def __init__(self, shape, dtype, device=0, kept=None):
        self.shape, self.dtype, self.is_cuda = tuple(shape), np.dtype(dtype), True
        self.nbytes, self.on, self.kept = int(np.prod(shape)) * self.dtype.itemsize, device, kept

    def data_ptr(self):
        return 0x1000

    def get_device(self):
        return self.on

    def is_contiguous(self):
        return True

    def stride(self):
        return tuple(np.cumprod((1, *self.shape[:0:-1]))[::-1].tolist())

    def record_stream(self, s):
        self.kept.append((id(self), s))


class Device:
    """torch's current device, and what is called under which."""

    def __init__(self, monkeypatch, lib, current):
        self.current, self.under = current, []
        monkeypatch.setattr(kc, "_is_torch", lambda a: isinstance(a, Tensorlike))
        monkeypatch.setattr(kc, "_torch_names", lambda: kc._TORCH)
        monkeypatch.setattr(kc, "_empty", lambda like, shape, dtype, stream=None: Tensorlike(
            shape, kc._NUMPY[dtype], like.on, like.kept))
        monkeypatch.setattr(kc, "_torch_device", lambda: self.current)
        monkeypatch.setattr(kc, "_raw_stream", lambda device: 16 + device)
        monkeypatch.setitem(sys.modules, "torch", types.SimpleNamespace(
            cuda=types.SimpleNamespace(device=self.switch), Tensor=Tensorlike))
        for name in ("work_bytes", "attend_bytes", "plan", "append", "attend", "read"):
            name = "grm_hip_kv_" + name
            setattr(lib, name, lambda *a, fn=getattr(lib, name), n=name: (
                self.under.append((n, self.current, a)), fn(*a))[1])

    @contextlib.contextmanager
    def switch(self, device):
        was, self.current = self.current, device
        yield
        self.current = was


def on_gpu(device, **kw):
    def T(shape, dtype):
        return Tensorlike(shape, dtype, kw.get(str(shape), device), kw.get("kept"))
    cache = g.KvCache(T((4, 2, 16, 64), np.int8), T((4, 2, 64, 16), np.int8),
                      T((4, 2), np.float32), T((4, 2), np.float32))
    batch = g.KvBatch(T((3,), np.int32), T((3,), np.int32), T((3, 4), np.int32), 16, tokens=3,
                      max_new=1, heads=4, kv_heads=2, free_list=T((9,), np.int32),
                      free_head=T((1,), np.int32))
    return T, cache, batch


def test_a_batch_is_kept_for_the_streams_that_read_it(lib, monkeypatch):
    """The schedule and the other arrays that a batch made are recorded for every
    stream that a call names, beside the one that they were made on."""
    kept = []
    Device(monkeypatch, lib, current=0)
    monkeypatch.setattr(kc, "_torch_stream", lambda a, on: ("stream", on))
    T, c, b = on_gpu(0, kept=kept)
    mine = {id(a) for a in (b.cu_new, b.slot_map, b.positions, b._work, b.free_head_out)}
    b.plan()
    b.plan(stream=16)
    assert not kept                                # where they were made
    b.plan(stream=7)
    assert {i for i, _ in kept} == mine and {s for _, s in kept} == {("stream", 7)}
    x = T((3, 2, 64), np.float32)
    c.append(b, x, x, stream=7)
    assert len(kept) == len(mine)                  # once is enough
    c.append(b, x, x, stream=8)
    assert kept[-1][1] == ("stream", 8)
    c.attend(b, T((3, 4, 64), np.float32), stream=0)
    assert {i for i, s in kept if s == ("stream", 0)} == mine


def test_calls_run_on_the_arrays_device(lib, monkeypatch):
    """Whatever device is current: sizes, launches and streams are those of the
    GPU that the arrays are on."""
    d = Device(monkeypatch, lib, current=0)
    T, cache, batch = on_gpu(1)
    batch.plan()
    cache.append(batch, T((3, 2, 64), np.float32), T((3, 2, 64), np.float32))
    cache.attend(batch, T((3, 4, 64), np.float32), return_lse=True)
    cache.read(T((3, 4), np.int32), T((3,), np.int32), T((4,), np.int32), 5)
    assert len(d.under) == 6 and d.current == 0
    for name, current, args in d.under:
        assert current == 1, name
        if not name.endswith("bytes"):
            assert args[-1] == 17, name            # that device's stream
    assert {batch.device, cache.device, batch.cu_new.get_device()} == {1}


def test_arrays_of_several_gpus_are_refused(lib, monkeypatch):
    d = Device(monkeypatch, lib, current=0)
    for other in ((3, 4), (9,), (4, 2)):
        with pytest.raises(ValueError, match="more than one GPU"):
            on_gpu(0, **{str(other): 1})
    T, cache, batch = on_gpu(0)
    _, far, _ = on_gpu(1)
    batch.plan()
    d.under.clear()
    f4, i4 = np.float32, np.int32
    kv, q, there = T((3, 2, 64), f4), T((3, 4, 64), f4), lambda s, t: Tensorlike(s, t, 1)
    for call in (lambda: cache.append(batch, there((3, 2, 64), f4), kv),
                 lambda: cache.append(batch, kv, there((3, 2, 64), f4)),
                 lambda: cache.attend(batch, there((3, 4, 64), f4)),
                 lambda: cache.attend(batch, q, out=there((3, 4, 64), f4)),
                 lambda: cache.attend(batch, q, lse=there((3, 4), f4)),
                 lambda: far.append(batch, kv, kv), lambda: far.attend(batch, q),
                 lambda: cache.read(T((3, 4), i4), there((3,), i4), T((4,), i4), 5),
                 lambda: far.read(T((3, 4), i4), T((3,), i4), T((4,), i4), 5),
                 lambda: batch.plan(stream=types.SimpleNamespace(device_index=1, cuda_stream=9))):
        with pytest.raises(ValueError, match="GPU 1"):
            call()
    assert not [u for u in d.under if not u[0].endswith("bytes")]


def test_device_arrays_of_another_gpu_than_the_current_are_refused(lib, monkeypatch):
    b, c = batch_of(), cache_of(64)
    monkeypatch.setattr(kc, "current_device", lambda: 1)
    for call in (b.plan, batch_of):
        with pytest.raises(ValueError, match="GPU 0, the current device is GPU 1"):
            call()
    monkeypatch.setattr(kc, "current_device", lambda: 0)
    b.plan()
    x = fake((3, 4, 64), np.float32)
    x.device = 1
    with pytest.raises(ValueError, match="GPU 1"):
        c.attend(b, x)


def test_values_that_require_a_gradient_are_refused(lib, monkeypatch):
    """There is no backward pass, and a result without one must not look like one."""
    Device(monkeypatch, lib, current=0)
    T, cache, batch = on_gpu(0)
    batch.plan()
    kv, q = T((3, 2, 64), np.float32), T((3, 4, 64), np.float32)
    kv2, q2 = T((3, 2, 64), np.float32), T((3, 4, 64), np.float32)
    kv2.requires_grad = q2.requires_grad = True
    sys.modules["torch"].is_grad_enabled = lambda: True
    for call in (lambda: cache.append(batch, kv2, kv), lambda: cache.append(batch, kv, kv2),
                 lambda: cache.attend(batch, q2), lambda: cache.attend(batch, q, out=q2)):
        with pytest.raises(ValueError, match="no backward"):
            call()
    sys.modules["torch"].is_grad_enabled = lambda: False
    cache.append(batch, kv2, kv2)
    cache.attend(batch, q2)


def test_the_free_list_goes_on_once_a_plan(lib):
    """A second advance would go back to the head before, whose blocks the plan
    has handed out; one before any plan, to memory that nobody has written."""
    b = batch_of(free_list=fake((9,), np.int32), free_head=fake((1,), np.int32))
    first, second = b.free_head, b.free_head_out
    with pytest.raises(ValueError, match="no plan"):
        b.advance()
    assert b.free_head is first
    b.plan().plan().advance()
    assert b.free_head is second and b._desc.free_head == second.data_ptr()
    with pytest.raises(ValueError, match="no plan"):
        b.advance()
    b.plan().advance()
    assert b.free_head is first


@pytest.mark.parametrize("name", ["tokens", "max_new", "heads", "kv_heads", "window",
                                  "block_tokens"])
def test_sizes_that_do_not_fit_are_refused(lib, name):
    """The descriptor's fields have 32 bits: 2^32 + 4 is not 4."""
    sizes = dict(tokens=3, max_new=1, heads=4, kv_heads=2, window=0, block_tokens=16)
    for off in (1 << 32, 1 << 31, -(1 << 32)):
        bad = {**sizes, name: sizes[name] + off}
        bs = bad.pop("block_tokens")
        with pytest.raises(ValueError, match=name):
            g.KvBatch(fake((3,), np.int32), fake((3,), np.int32), fake((3, 4), np.int32), bs, **bad)
    with pytest.raises(ValueError, match="rows"):
        cache_of(64).read(fake((3, 4), np.int32), fake((3,), np.int32), fake((4,), np.int32), -1)
