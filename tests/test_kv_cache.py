"""What the 8-bit key/value cache refuses, and its host laws (CPU only: no
kernel is launched)."""

import ctypes

import numpy as np
import pytest

import graftrepository_amd as g
from graftrepository_amd import kv_cache as kc
from oracle import kv as law



def fake(shape, dtype):
    a = g.payload.DeviceArray.__new__(g.payload.DeviceArray)
    a.shape, a.dtype = tuple(shape), np.dtype(dtype)
    a.size = int(np.prod(shape))
    a.nbytes = a.size * a.dtype.itemsize
    a.ptr = 0x1000
    a.close = lambda: None
    return a


def cache_desc(**kw):
    d = kc._CacheDesc()
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        setattr(d, name, 0x1000)
    d.blocks, d.block_tokens, d.kv_heads, d.head_dim = 4, 16, 2, 64
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def batch_desc(**kw):
    d = kc._BatchDesc()
    for name in ("ctx_lens", "new_lens", "block_table", "cu_new", "work"):
        setattr(d, name, 0x1000)
    d.work_bytes = 1 << 40
    d.requests, d.table_width, d.tokens, d.max_new = 3, 4, 3, 1
    d.block_tokens, d.heads, d.kv_heads, d.window = 16, 4, 2, 0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_BATCH = [
    (dict(block_tokens=24), b"block_tokens"), (dict(block_tokens=0), b"block_tokens"),
    (dict(heads=5), b"multiple"), (dict(kv_heads=0), b"multiple"), (dict(heads=0), b"multiple"),
    (dict(heads=65536, kv_heads=2), b"65535"),
    (dict(requests=-1), b"negative"), (dict(tokens=-1), b"negative"),
    (dict(max_new=-2), b"negative"), (dict(window=-1), b"negative"),
    (dict(table_width=-1), b"negative"), (dict(tokens=(1 << 31) - 1), b"too large"),
    (dict(ctx_lens=None), b"null"), (dict(work=None), b"null"), (dict(cu_new=None), b"null"),
    (dict(block_table=None), b"block table"), (dict(work=0x1008), b"aligned"),
    (dict(free_list=0x1000), b"both heads"),
    (dict(free_list=0x1000, free_head=0x1000), b"both heads"),
    (dict(free_list=0x1000, free_head=0x1000, free_head_out=0x1000), b"must not be"),
    (dict(free_head=0x1000, free_head_out=0x2000, free_count=3), b"null free list"),
    (dict(free_list=0x1000, free_head=0x1000, free_head_out=0x2000, free_count=1 << 31),
     b"too long"),
]


@pytest.mark.parametrize("change,word", BAD_BATCH)
def test_a_bad_batch_is_refused(change, word):
    lib = g.load()
    d = batch_desc(**change)
    assert lib.grm_hip_kv_plan(ctypes.byref(d), None) == -1
    assert word in lib.grm_hip_last_error()


BAD_CACHE = [
    (dict(head_dim=24), b"head_dim"), (dict(head_dim=272), b"head_dim"),
    (dict(head_dim=0), b"head_dim"), (dict(block_tokens=48), b"block_tokens"),
    (dict(blocks=0), b"block count"), (dict(blocks=1 << 31), b"block count"),
    (dict(kv_heads=0), b"kv_heads"), (dict(k_codes=None), b"null"), (dict(v_scales=None), b"null"),
    (dict(v_codes=0x1004), b"aligned"), (dict(kv_heads=4), b"differ"),
    (dict(block_tokens=32), b"differ"),
]


@pytest.mark.parametrize("change,word", BAD_CACHE)
def test_a_bad_cache_is_refused(change, word):
    lib = g.load()
    c, b = cache_desc(**change), batch_desc()
    assert lib.grm_hip_kv_append(ctypes.byref(c), ctypes.byref(b), 0x1000, 0x1000, 0, 128, 64, 128,
                                 64, None) == -1
    assert word in lib.grm_hip_last_error()


def test_bad_call_arguments_are_refused():
    lib = g.load()
    c, b = cache_desc(), batch_desc()
    rc, rb = ctypes.byref(c), ctypes.byref(b)
    out = ctypes.c_uint64()
    assert lib.grm_hip_kv_work_bytes(rb, None) == -1
    assert lib.grm_hip_kv_work_bytes(None, ctypes.byref(out)) == -1
    assert lib.grm_hip_kv_attend_bytes(rc, rb, None) == -1
    # append: a type that is no float, null keys
    assert lib.grm_hip_kv_append(rc, rb, 0x1000, 0x1000, 3, 128, 64, 128, 64, None) == -1
    assert lib.grm_hip_kv_append(rc, rb, None, 0x1000, 0, 128, 64, 128, 64, None) == -1

    def attend(q=0x1000, dtype=1, qt=256, qh=64, out=0x1000, ot=256, oh=64, scale=1.0):
        return lib.grm_hip_kv_attend(rc, rb, q, dtype, qt, qh, out, ot, oh, None, scale, None, 0,
                                     None)
    for kw in (dict(q=None), dict(out=None), dict(q=0x1002), dict(out=0x1008), dict(dtype=3),
               dict(qt=257), dict(qh=60), dict(ot=4), dict(oh=66), dict(scale=float("nan")),
               dict(scale=float("inf"))):
        assert attend(**kw) == -1, kw
    read = lib.grm_hip_kv_read
    assert read(rc, 0x1000, 4, 3, 0x1000, 0x1000, 5, 3, 0x1000, 0x1000, None) == -1
    assert read(rc, 0x1000, 4, 0, 0x1000, 0x1000, 5, 0, 0x1000, 0x1000, None) == -1
    assert read(rc, None, 4, 3, 0x1000, 0x1000, 5, 0, 0x1000, 0x1000, None) == -1
    assert read(rc, 0x1000, 4, 3, 0x1000, None, 5, 0, 0x1000, 0x1000, None) == -1
    assert read(rc, 0x1000, 4, 3, 0x1000, 0x1000, 5, 0, 0x1004, 0x1000, None) == -1


def test_python_checks_shapes_types_and_memory():
    i8, f4, i4 = np.int8, np.float32, np.int32
    good = dict(k_codes=fake((4, 2, 16, 64), i8), v_codes=fake((4, 2, 64, 16), i8),
                k_scales=fake((4, 2), f4), v_scales=fake((4, 2), f4))
    cache = g.KvCache(**good)
    assert (cache.blocks, cache.block_tokens, cache.kv_heads, cache.head_dim) == (4, 16, 2, 64)
    for change in (dict(k_codes=fake((4, 2, 16, 64), np.uint8)),
                   dict(v_codes=fake((4, 2, 16, 64), i8)),
                   dict(k_scales=fake((4, 2, 1), f4)), dict(v_scales=fake((4, 2), np.float16)),
                   dict(k_codes=fake((4, 2, 20, 64), i8), v_codes=fake((4, 2, 64, 20), i8)),
                   dict(k_codes=fake((4, 2, 16, 40), i8), v_codes=fake((4, 2, 40, 16), i8)),
                   dict(k_codes=np.zeros((4, 2, 16, 64), i8))):
        with pytest.raises(ValueError):
            g.KvCache(**{**good, **change})
    with pytest.raises(ValueError):
        cache.read(fake((3, 4), i4), fake((3,), i4), fake((3,), i4), 5)
    with pytest.raises(ValueError):
        cache.read(fake((3, 4), i4), fake((3,), i4), fake((4,), i4), 5, dtype="i8")
    with pytest.raises(ValueError):
        kc._rows(fake((5, 2, 64), i8), "q", (5, 2, 64))
    with pytest.raises(ValueError):
        kc._rows(fake((5, 2, 64), f4), "q", (5, 4, 64))


def test_torch_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="GPU"):
        g.KvCache(torch.zeros((4, 2, 16, 64), dtype=torch.int8),
                  torch.zeros((4, 2, 64, 16), dtype=torch.int8), torch.zeros(4, 2),
                  torch.zeros(4, 2))


# --------------------------------------------------------- the laws themselves

def test_append_law_rounds_within_half_a_step_and_keeps_what_a_block_held():
    rng = np.random.default_rng(0)
    codes = np.zeros((4, 2, 16, 8), np.int8)
    scales = np.full((4, 2), np.nan, np.float32)
    table = np.array([[2, 0]], np.int32)
    x = rng.standard_normal((20, 2, 8)).astype(np.float32)
    law.append(codes, scales, x[:5], [0], [5], table, False)
    first = scales[2].copy()
    law.append(codes, scales, 4 * x[5:], [5], [15], table, False)
    assert (scales[2] >= first).all() and np.isnan(scales[1]).all()
    got = law.values(codes, scales, table[0], False)[:20]
    step = np.repeat(scales[table[0]], 16, 0)[:20, :, None]
    want = np.concatenate([x[:5], 4 * x[5:]])
    # kept codes were rounded twice: half a step of the first scale, half of
    # the second
    assert (np.abs(got - want) <= step * (1.0 + 1e-5)).all()
    assert (np.abs(got - want)[5:] <= step[5:] * 0.5 * (1 + 1e-5)).all()


def test_attend_law_against_differences():
    # d lse / d q = softmax_scale * sum_j p_j k_j: with values that are the
    # keys, the output is that gradient
    rng = np.random.default_rng(1)
    hd, bs, n = 16, 16, 29
    k = rng.integers(-127, 128, (2, 1, bs, hd)).astype(np.int8)
    v = np.ascontiguousarray(k.transpose(0, 1, 3, 2))
    s = np.array([[0.01], [0.02]], np.float32)
    table = np.array([[1, 0]], np.int32)
    q = rng.standard_normal((1, 1, hd))
    run = lambda q: law.attend(q, k, v, s, s, [n - 1], [1], table, 0.25)  # noqa: E731
    out = run(q)[0][0, 0]
    for d in range(hd):
        step = np.zeros_like(q)
        step[0, 0, d] = 1e-5
        slope = (run(q + step)[1] - run(q - step)[1])[0, 0] / 2e-5
        assert abs(slope - 0.25 * out[d]) < 1e-8


def test_plan_law_by_hand():
    table = np.full((3, 3), -1)
    table[0, 0] = 9
    t, cu, slots, pos, head = law.plan([15, 0, 4], [2, 17, 0], table, 16, 20, [5, 6, 7, 8], 0)
    assert t.tolist() == [[9, 5, -1], [6, 7, -1], [-1, -1, -1]]
    assert cu.tolist() == [0, 2, 19, 19] and head == 3
    assert slots[:3].tolist() == [9 * 16 + 15, 5 * 16, 6 * 16] and slots[18:].tolist() == [112, -1]
    assert pos.tolist() == [15, 16] + list(range(17)) + [-1]
