"""What rotary positions and the latent cache refuse (CPU only: no kernel is
launched)."""

import ctypes
import math

import numpy as np
import pytest

import graftrepository_amd as g
from graftrepository_amd import rotary as rt
from oracle import latent as law
from tests.test_kv_cache import batch_desc, cache_desc, fake


@pytest.mark.parametrize("kw", [
    dict(dim=0), dict(dim=7), dict(dim=258), dict(dim=-2), dict(layout="pairs"), dict(scaling="far"),
    dict(base=1.0), dict(base=float("inf")), dict(factor=0.0), dict(factor=float("nan")),
    dict(trained=0), dict(fast=1.0, slow=2.0), dict(slow=0.0), dict(magnitude=0.0),
    dict(magnitude=float("nan")), dict(scaling="factors"), dict(scaling="factors", factors=[1.0]),
    dict(scaling="factors", factors=[0.01] * 32), dict(dim=2, scaling="base", factor=2.0)])
def test_a_bad_rotary_is_refused(kw):
    with pytest.raises(ValueError):
        g.Rotary(**{"dim": 64, **kw})


def test_frequencies_by_hand():
    assert g.Rotary(4, base=100.0).frequencies == pytest.approx([1.0, 0.1])
    assert g.Rotary(4, base=100.0, scaling="linear", factor=4).frequencies == pytest.approx([0.25, 0.025])
    # base 100 * 4^(4/2) = 1600
    assert g.Rotary(4, base=100.0, scaling="base", factor=4).frequencies == pytest.approx([1.0, 0.025])
    yarn = g.Rotary(64, scaling="yarn", factor=8)
    plain = g.Rotary(64)
    assert yarn.frequencies[0] == plain.frequencies[0]
    assert yarn.frequencies[-1] == pytest.approx(plain.frequencies[-1] / 8)
    assert yarn.magnitude == pytest.approx(0.1 * math.log(8) + 1)
    smooth = g.Rotary(64, scaling="smooth", factor=8, trained=8192, slow=1, fast=4)
    for f, p in zip(smooth.frequencies, plain.frequencies):
        turns = p * 8192 / (2 * math.pi)
        want = p if turns > 4 else p / 8 if turns < 1 else None
        assert want is None or f == pytest.approx(want)
        assert p / 8 * (1 - 1e-12) <= f <= p * (1 + 1e-12)


BAD_DESC = [(dict(dim=3), b"even"), (dict(dim=0), b"even"), (dict(dim=258), b"even"),
            (dict(dim=128), b"more channels"), (dict(layout=2), b"layout"),
            (dict(magnitude=0.0), b"magnitude"), (dict(magnitude=float("nan")), b"magnitude"),
            (dict(magnitude=float("inf")), b"magnitude"), (dict(turn=2.0), b"frequency"),
            (dict(turn=float("nan")), b"frequency")]


def rotary_desc(**kw):
    d = rt._RotaryDesc()
    d.dim, d.magnitude = 64, 1.0
    d.turns[:] = [0.01] * 128
    for k, v in kw.items():
        if k == "turn":
            d.turns[5] = v
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,word", BAD_DESC)
def test_a_bad_descriptor_is_refused(change, word):
    lib = g.load()
    d = rotary_desc(**change)
    assert lib.grm_hip_rotate(ctypes.byref(d), 0x1000, 0, 64, 64, 0x2000, 64, 64, 0x1000, 4, 1, 64,
                              0, None) == -1
    assert word in lib.grm_hip_last_error()
    c, b = cache_desc(), batch_desc(positions=0x1000)
    assert lib.grm_hip_kv_append_turned(ctypes.byref(c), ctypes.byref(b), ctypes.byref(d), 0x1000,
                                        0x1000, 0, 128, 64, 128, 64, None) == -1
    assert word in lib.grm_hip_last_error()


def test_bad_calls_are_refused():
    lib = g.load()
    d = ctypes.byref(rotary_desc())

    def rotate(rotary=d, x=0x1000, dtype=0, out=0x2000, xt=64, ot=64, pos=0x1000, n=4, heads=1,
               hd=64, start=0):
        return lib.grm_hip_rotate(rotary, x, dtype, xt, 64, out, ot, 64, pos, n, heads, hd, start,
                                  None)
    for kw in (dict(rotary=None), dict(x=None), dict(out=None), dict(pos=None), dict(dtype=3),
               dict(heads=0), dict(heads=65536), dict(hd=0), dict(hd=32), dict(start=-1),
               dict(start=65), dict(start=1), dict(n=1 << 31), dict(out=0x1000, ot=128)):
        assert rotate(**kw) == -1, kw
    assert rotate(n=0) == 0
    c, b = ctypes.byref(cache_desc()), batch_desc()
    assert lib.grm_hip_kv_append_turned(c, ctypes.byref(b), d, 0x1000, 0x1000, 0, 128, 64, 128, 64,
                                        None) == -1     # no positions
    assert b"positions" in lib.grm_hip_last_error()
    assert lib.grm_hip_kv_append_turned(c, ctypes.byref(b), None, 0x1000, 0x1000, 0, 128, 64, 128,
                                        64, None) == -1


def test_python_checks_of_apply():
    rotary = g.Rotary(32)
    x, pos = fake((4, 2, 64), np.float32), fake((4,), np.int32)
    for args, kw in (((fake((4, 64), np.float32), pos), {}), ((x, fake((5,), np.int32)), {}),
                     ((x, fake((4,), np.int64)), {}), ((x, pos), dict(start=33)),
                     ((x, pos), dict(start=-1)), ((fake((4, 2, 16), np.float32), pos), {}),
                     ((x, pos), dict(out=fake((4, 2, 64), np.float16))),
                     ((x, pos), dict(out=fake((4, 2, 32), np.float32))),
                     ((fake((4, 2, 64), np.int8), pos), {})):
        with pytest.raises(ValueError):
            rotary.apply(*args, **kw)


def test_values_that_require_a_gradient_are_refused():
    torch = pytest.importorskip("torch")
    x = torch.zeros((2, 1, 64), requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        g.Rotary(64).apply(x, torch.zeros(2, dtype=torch.int32))


def test_the_law_against_complex_numbers_and_its_inverse():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 2, 12))
    f = [0.3, 0.02, 0.7]
    pos = [0, 3, 100, 7, 5]
    for layout in ("half", "interleaved"):
        y, _ = law.turned(x, pos, f, 1.5, layout, 2)
        pairs = (slice(2, 5), slice(5, 8)) if layout == "half" else (slice(2, 8, 2), slice(3, 8, 2))
        z = (x[..., pairs[0]] + 1j * x[..., pairs[1]]) * 1.5 * np.exp(
            1j * np.array(pos)[:, None, None] * np.array(f))
        assert np.allclose(y[..., pairs[0]], z.real) and np.allclose(y[..., pairs[1]], z.imag)
        assert (y[..., :2] == x[..., :2]).all() and (y[..., 8:] == x[..., 8:]).all()
        assert np.allclose(law.turned(y, pos, f, 1.5, layout, 2, inverse=True)[0], x)


# ------------------------------------------------------------ latent cache

def latent_desc(**kw):
    from graftrepository_amd import latent as lt
    d = lt._LatentDesc()
    d.rows, d.blocks, d.block_tokens, d.rank, d.rope, d.dtype = 0x1000, 4, 16, 64, 32, 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def one_head(**kw):
    return batch_desc(**{**dict(heads=4, kv_heads=1, slot_map=0x1000, positions=0x1000), **kw})


BAD_LATENT = [(dict(rows=None), b"null"), (dict(rows=0x1008), b"aligned"), (dict(blocks=0), b"block count"),
              (dict(blocks=1 << 31), b"block count"), (dict(block_tokens=48), b"block_tokens"),
              (dict(block_tokens=32), b"differ"), (dict(rank=0), b"rank"), (dict(rank=520), b"rank"),
              (dict(rank=1024), b"rank"), (dict(rope=8), b"rope"), (dict(rope=144), b"rope"),
              (dict(rope=-16), b"rope"), (dict(dtype=0), b"BF16"), (dict(dtype=3), b"BF16")]


@pytest.mark.parametrize("change,word", BAD_LATENT)
def test_a_bad_latent_cache_is_refused(change, word):
    lib = g.load()
    c, b = latent_desc(**change), one_head()
    assert lib.grm_hip_latent_append(ctypes.byref(c), ctypes.byref(b), None, 0x1000, 0x1000, 0, 64,
                                     32, None) == -1
    assert word in lib.grm_hip_last_error()


def test_bad_latent_calls_are_refused():
    lib = g.load()
    c = ctypes.byref(latent_desc())

    def append(batch=None, rotary=None, latents=0x1000, keys=0x1000, dtype=0):
        return lib.grm_hip_latent_append(c, ctypes.byref(batch or one_head()), rotary, latents, keys,
                                         dtype, 64, 32, None)
    odd = rotary_desc(dim=24)
    for kw in (dict(batch=one_head(kv_heads=2)), dict(batch=one_head(slot_map=None)),
               dict(batch=one_head(positions=None), rotary=ctypes.byref(rotary_desc(dim=32))),
               dict(latents=None), dict(keys=None), dict(dtype=3),
               dict(rotary=ctypes.byref(odd)), dict(rotary=ctypes.byref(rotary_desc(dim=64)))):
        assert append(**kw) == -1, kw
    read = lib.grm_hip_latent_read
    assert read(c, 0x1000, 4, 3, 0x1000, 0x1000, 5, 3, 0x1000, None) == -1
    assert read(c, 0x1000, 4, 0, 0x1000, 0x1000, 5, 0, 0x1000, None) == -1
    assert read(c, None, 4, 3, 0x1000, 0x1000, 5, 0, 0x1000, None) == -1
    assert read(c, 0x1000, 4, 3, 0x1000, None, 5, 0, 0x1000, None) == -1
    assert read(c, 0x1000, 4, 3, 0x1000, 0x1000, 5, 0, 0x1004, None) == -1
    assert read(c, 0x1000, 4, 3, 0x1000, 0x1000, 5, 0, None, None) == -1
    assert read(c, 0x1000, -1, 3, 0x1000, 0x1000, 5, 0, 0x1000, None) == -1
    assert read(c, 0x1000, 4, 3, 0x1000, 0x1000, 0, 0, None, None) == 0


def test_python_checks_of_a_latent_cache():
    for shape, dtype, rank in (((4, 16, 96), np.float32, 64), ((4, 16), np.float16, 64),
                               ((4, 20, 96), np.float16, 64), ((4, 16, 96), np.float16, 60),
                               ((4, 16, 96), np.float16, 112), ((4, 16, 700), np.float16, 528),
                               ((4, 16, 100), np.float16, 64), ((4, 16, 256), np.float16, 64)):
        with pytest.raises(ValueError):
            g.LatentCache(fake(shape, dtype), rank)
    c = g.LatentCache(fake((4, 16, 96), np.float16), 64)
    assert (c.blocks, c.block_tokens, c.rank, c.rope, c.dtype) == (4, 16, 64, 32, "f16")
    with pytest.raises(ValueError):
        c.read(fake((3, 4), np.int32), fake((3,), np.int32), fake((3,), np.int32), 5)
    with pytest.raises(ValueError):
        c.read(fake((3, 4), np.int32), fake((3,), np.int32), fake((4,), np.int32), 5, dtype="i8")


def test_bad_attention_calls_are_refused():
    lib = g.load()
    c, out = ctypes.byref(latent_desc()), ctypes.c_uint64()
    b = one_head()
    rb = ctypes.byref(b)
    assert lib.grm_hip_latent_work_bytes(rb, None) == -1
    assert lib.grm_hip_latent_work_bytes(None, ctypes.byref(out)) == -1
    assert lib.grm_hip_latent_attend_bytes(c, rb, None) == -1
    assert lib.grm_hip_latent_plan(rb, None, 1 << 40, None) == -1
    assert lib.grm_hip_latent_plan(rb, 0x1008, 1 << 40, None) == -1
    assert lib.grm_hip_latent_plan(ctypes.byref(one_head(new_lens=None)), 0x1000, 1 << 40, None) == -1

    def attend(cache=c, batch=rb, work=0x1000, q=0x1000, qt=384, qh=96, o=0x2000, ot=256, oh=64,
               scale=1.0):
        return lib.grm_hip_latent_attend(cache, batch, work, 1 << 40, q, qt, qh, o, ot, oh, None,
                                         scale, None, 0, None)
    for kw in (dict(q=None), dict(o=None), dict(q=0x1002), dict(o=0x2008), dict(qt=385), dict(qh=100),
               dict(ot=4), dict(oh=66), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(batch=ctypes.byref(one_head(kv_heads=2))), dict(cache=None), dict(batch=None)):
        assert attend(**kw) == -1, kw


def test_python_checks_of_latent_batches():
    ints = [fake((3,), np.int32), fake((3,), np.int32), fake((3, 4), np.int32)]
    with pytest.raises(ValueError, match="kv_heads"):
        g.KvBatch(*ints, 16, tokens=3, max_new=1, heads=4, kv_heads=2, latent=True)


def test_bad_expanded_calls_are_refused():
    lib = g.load()
    c = ctypes.byref(latent_desc())

    def expand(cache=c, weight=0x1000, heads=4, key=64, value=64, table=0x1000, width=4, requests=3,
               starts=0x1000, cu=0x1000, rows=5, k=0x1000, v=0x1000):
        return lib.grm_hip_latent_expand(cache, weight, heads, key, value, table, width, requests,
                                         starts, cu, rows, k, v, None)
    for kw in (dict(cache=None), dict(weight=None), dict(weight=0x1008), dict(heads=0),
               dict(heads=65536), dict(key=0), dict(key=12), dict(key=520), dict(value=0),
               dict(value=12), dict(value=520), dict(table=None), dict(requests=0), dict(starts=None),
               dict(cu=None), dict(k=None), dict(v=0x1004), dict(rows=1 << 31), dict(width=-1),
               dict(rows=1 << 29, heads=65535)):
        assert expand(**kw) == -1, kw
    assert expand(rows=0) == 0

    def rows(batch=None, work=0x1000, dtype=1, dk=64, dv=64, q=0x1000, k=0x1000, v=0x1000, stride=64,
             n=5, cu=0x1000, out=0x1000, scale=1.0):
        b = batch or one_head()
        return lib.grm_hip_rows_attend(ctypes.byref(b), work, 1 << 40, dtype, dk, dv, q, 256, 64, k,
                                       stride, 64, v, 256, 64, n, cu, None, out, 256, 64, None, scale,
                                       None, 0, None)
    for kw in (dict(batch=one_head(kv_heads=2)), dict(work=None), dict(work=0x1008), dict(dtype=0),
               dict(dk=0), dict(dk=12), dict(dk=520), dict(dv=4), dict(dv=1024), dict(q=None),
               dict(k=None), dict(v=None), dict(cu=None), dict(out=None), dict(q=0x1002),
               dict(k=0x1008), dict(stride=60), dict(n=1 << 31), dict(scale=float("nan"))):
        assert rows(**kw) == -1, kw


def test_python_checks_of_the_expanded_form():
    c = g.LatentCache(fake((4, 16, 96), np.float16), 64)
    at = (fake((3, 4), np.int32), fake((3,), np.int32), fake((4,), np.int32), 5)
    for weight, key in ((fake((4, 64), np.float16), 32), (fake((4, 64, 64), np.float32), 32),
                        (fake((4, 64, 32), np.float16), 32), (fake((4, 64, 64), np.float16), 64),
                        (fake((4, 64, 64), np.float16), 0)):
        with pytest.raises(ValueError):
            c.expand(weight, key, *at)


def test_rows_that_are_one_another_are_not_turned_in_place():
    lib = g.load()
    d = ctypes.byref(rotary_desc())
    for strides in ((0, 64), (128, 0)):     # a row given to all tokens, a head to all heads
        assert lib.grm_hip_rotate(d, 0x1000, 0, *strides, 0x1000, *strides, 0x1000, 4, 2, 64, 0,
                                  None) == -1
        assert b"memory" in lib.grm_hip_last_error()
    # a row of more values than an index holds
    assert lib.grm_hip_rotate(d, 0x1000, 0, 64, 64, 0x2000, 64, 64, 0x1000, 4, 65535, 65536, 0,
                              None) == -1
