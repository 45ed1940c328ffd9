"""Rotary positions on the GPU against fp64, and keys turned on their way into
the caches against the two steps one after the other, bit for bit."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch, KvCache, LatentCache, Rotary  # noqa: E402
from graftrepository_amd.payload import DeviceArray  # noqa: E402
from oracle import latent as law  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(dtype) if dtype is not None else t


def host(t):
    return t.double().cpu().numpy()


def check(got, x, positions, rotary, start, name, inverse=False):
    want, mass = law.turned(host(x), positions, rotary.frequencies, rotary.magnitude, rotary.layout,
                            start, inverse)
    bound = law.turned_bound(want, mass, name)
    seen = np.asarray(positions) >= 0
    off = np.abs(host(got) - want)
    assert (off <= bound)[seen].all(), (off / np.maximum(bound, 1e-300))[seen].max()


SHAPES = [
    # tokens, heads, head_dim, start, dim
    (1, 1, 64, 0, 64), (3, 5, 128, 0, 128), (7, 40, 96, 64, 32), (130, 2, 256, 0, 64),
    (33, 1, 256, 0, 256), (5, 3, 192, 128, 64), (1, 128, 192, 128, 64), (2048, 1, 64, 0, 64),
    # no whole units of sixteen
    (4, 3, 10, 2, 6), (9, 2, 24, 0, 24), (2, 7, 2, 0, 2), (6, 2, 40, 4, 32), (3, 300, 20, 0, 8),
]


@pytest.mark.parametrize("tokens,heads,hd,start,dim", SHAPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
def test_rotation_matches_the_law(hip_lib, tokens, heads, hd, start, dim, layout, name):
    rng = np.random.default_rng(tokens + hd + dim)
    x = dev(rng.standard_normal((tokens, heads, hd)), TYPES[name])
    positions = rng.integers(0, 200_000, tokens).astype(np.int32)
    positions[::3] = 0
    rotary = Rotary(dim, layout=layout, scaling="yarn", factor=8.0)
    got = rotary.apply(x, dev(positions), start=start)
    check(got, x, positions, rotary, start, name)
    back = rotary.apply(x, dev(positions), start=start, inverse=True)
    check(back, x, positions, rotary, start, name, inverse=True)
    mine = x.clone()
    assert rotary.apply(mine, dev(positions), start=start, out=mine) is mine
    assert torch.equal(mine, got)


def test_far_positions_keep_their_angles(hip_lib):
    rng = np.random.default_rng(0)
    positions = np.array([0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 30 - 257, 2 ** 31 - 1], np.int32)
    x = dev(rng.standard_normal((6, 2, 128)), torch.float32)
    rotary = Rotary(128)
    check(rotary.apply(x, dev(positions)), x, positions, rotary, 0, "f32")


@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4), dict(scaling="base", factor=8),
                                dict(scaling="yarn", factor=40, magnitude=0.7),
                                dict(scaling="smooth", factor=8, trained=8192, slow=1, fast=4),
                                dict(scaling="factors", factors=[1 + 0.1 * i for i in range(32)])])
def test_scalings_turn_by_their_frequencies(hip_lib, kw):
    rng = np.random.default_rng(1)
    rotary = Rotary(64, base=500_000.0, **kw)
    positions = rng.integers(0, 100_000, 50).astype(np.int32)
    x = dev(rng.standard_normal((50, 3, 80)), torch.float32)
    check(rotary.apply(x, dev(positions), start=16), x, positions, rotary, 16, "f32")


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strides_and_rows_of_no_token(hip_lib, name, offset):
    rng = np.random.default_rng(2)
    whole = dev(rng.standard_normal((9, 4, 80 + offset)), TYPES[name])
    x = whole[:, 1:, offset:offset + 64]
    positions = np.array([5, -1, 7, 0, -1, 99, 1000, 3, -1], np.int32)
    rotary = Rotary(32, layout="interleaved")
    base = torch.full((9, 3, 70), 7.0, device="cuda", dtype=TYPES[name])
    out = base[..., 3:67] if offset == 1 else base[..., :64]
    rotary.apply(x, dev(positions), start=16, out=out)
    check(out, x, positions, rotary, 16, name)
    assert (out[torch.from_numpy(positions < 0).cuda()] == 7).all()
    if offset == 1:
        assert (base[..., :3] == 7).all() and (base[..., 67:] == 7).all()


def test_device_arrays_and_no_tokens(hip_lib):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 2, 32)).astype(np.float32)
    positions = np.arange(4, dtype=np.int32)
    rotary = Rotary(32)
    got = rotary.apply(DeviceArray.from_host(x), DeviceArray.from_host(positions))
    want = rotary.apply(dev(x), dev(positions))
    np.testing.assert_array_equal(got.to_host(), want.cpu().numpy())
    empty = torch.empty((0, 2, 32), device="cuda")
    assert rotary.apply(empty, torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 2, 32)


def test_values_that_are_not_finite_stay_in_their_pairs(hip_lib):
    x = torch.ones((1, 1, 64), device="cuda")
    x[0, 0, 5] = float("nan")
    x[0, 0, 40] = float("inf")
    got = Rotary(64).apply(x, torch.tensor([3], dtype=torch.int32, device="cuda"))[0, 0].cpu()
    bad = [i for i in range(64) if not math.isfinite(got[i])]
    assert bad == [5, 8, 37, 40]


# -------------------------------------------------- turned on their way in

def batch_of(ctx, new, bs, heads=2, kv_heads=2, extra=0, seed=0, **kw):
    rng = np.random.default_rng(seed)
    total = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    width = max(total) + 1
    pool = sum(total) + 2
    ids = rng.permutation(pool).astype(np.int32)
    table = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for r, t in enumerate(total):
        table[r, :t] = ids[at:at + t]
        at += t
    b = KvBatch(dev(np.array(ctx, np.int32)), dev(np.array(new, np.int32)), dev(table), bs,
                tokens=sum(new) + extra, max_new=max(new), heads=heads, kv_heads=kv_heads, **kw)
    return b.plan(), table, pool


APPENDS = [
    # ctx, new, kv, head_dim, dim, block
    ([0], [1], 1, 16, 16, 16), ([7, 0, 31], [1, 3, 2], 2, 64, 64, 16),
    ([100, 0, 5], [300, 17, 1], 2, 128, 128, 32), ([0, 63], [200, 70], 4, 256, 128, 128),
    ([3], [140], 1, 256, 256, 128), ([9, 64], [65, 1], 3, 96, 32, 64), ([2], [50], 2, 80, 80, 32),
    ([11, 0], [5, 30], 2, 48, 6, 16), ([40], [33], 1, 112, 20, 64),
]


@pytest.mark.parametrize("ctx,new,kv,hd,dim,bs", APPENDS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("aligned", [True, False])
def test_turned_append_is_rotation_then_append(hip_lib, ctx, new, kv, hd, dim, bs, layout, name,
                                               aligned):
    rng = np.random.default_rng(hd + dim)
    extra = 2
    b, table, pool = batch_of(ctx, new, bs, kv, kv, extra=extra)
    caches = []
    k0 = rng.integers(-127, 128, (pool, kv, bs, hd)).astype(np.int8)
    v0 = rng.integers(-127, 128, (pool, kv, hd, bs)).astype(np.int8)
    s0 = np.exp(rng.standard_normal((2, pool, kv)) - 4).astype(np.float32)
    for _ in range(2):
        caches.append(KvCache(dev(k0), dev(v0), dev(s0[0]), dev(s0[1])))
    n = sum(new) + extra
    k = dev(rng.standard_normal((n, kv, hd + 1)), TYPES[name])
    k = k[..., 1:] if not aligned else k[..., :hd].contiguous()
    v = dev(rng.standard_normal((n, kv, hd)), TYPES[name])
    rotary = Rotary(dim, layout=layout)
    caches[0].append(b, k, v, rotary=rotary)
    # the same in two steps, in fp32
    caches[1].append(b, rotary.apply(k.float(), b.positions), v.float())
    for a in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(caches[0], a), getattr(caches[1], a)), a


def test_a_key_that_is_not_finite_makes_its_block_so(hip_lib):
    b, table, pool = batch_of([0], [20], 16, 1, 1)
    cache = KvCache.empty(pool, 16, 1, 64)
    k = torch.ones((20, 1, 64), device="cuda")
    k[3, 0, 7] = float("inf")
    cache.append(b, k, torch.ones_like(k), rotary=Rotary(64))
    scales = cache.k_scales.to_host()
    assert np.isnan(scales[table[0, 0], 0]) and np.isfinite(scales[table[0, 1], 0])


LATENTS = [
    # ctx, new, rank, rope, dim, block
    ([0], [1], 512, 64, 64, 64), ([5, 0, 100], [1, 33, 200], 256, 32, 32, 16),
    ([0, 17], [130, 1], 16, 16, 16, 128), ([3], [40], 48, 128, 64, 32), ([1], [9], 80, 0, 0, 16),
]


@pytest.mark.parametrize("ctx,new,rank,rope,dim,bs", LATENTS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kept", ["bf16", "f16"])
@pytest.mark.parametrize("aligned", [True, False])
def test_latent_append_and_read(hip_lib, ctx, new, rank, rope, dim, bs, layout, name, kept, aligned):
    rng = np.random.default_rng(rank + rope)
    extra = 3
    b, table, pool = batch_of(ctx, new, bs, 4, 1, extra=extra)
    rows = dev(rng.standard_normal((pool, bs, rank + rope)), TYPES[kept])
    before = rows.clone()
    cache = LatentCache(rows, rank)
    n = sum(new)
    c = dev(rng.standard_normal((n + extra, rank + 1)), TYPES[name])
    c = c[:, 1:] if not aligned else c[:, :rank].contiguous()
    p = dev(rng.standard_normal((n + extra, rope)), TYPES[name]) if rope else None
    rotary = Rotary(dim, layout=layout) if dim else None
    cache.append(b, c, p, rotary=rotary)
    made = c.float()
    if rope:
        key = p.float()
        if rotary:
            key = rotary.apply(key[:, None].contiguous(), b.positions)[:, 0]
        made = torch.cat([made, key], 1)
    made = made[:n].to(TYPES[kept])
    slots = b.slot_map[:n].long()
    want = before.view(-1, rank + rope).clone()
    want[slots] = made
    assert torch.equal(rows.view(-1, rank + rope), want)
    # read back: everything the requests hold, and positions without a block
    starts = dev(np.array([max(0, c - 3) for c in ctx], np.int32))
    count = [c + m - max(0, c - 3) for c, m in zip(ctx, new)]
    count[-1] += 2 * bs
    cu = dev(np.concatenate([[0], np.cumsum(count)]).astype(np.int32))
    for out in ("f32", "bf16", "f16"):
        got = cache.read(dev(table), starts, cu, sum(count), dtype=out)
        at = 0
        for r in range(len(ctx)):
            first = max(0, ctx[r] - 3)
            for i in range(count[r]):
                j = (first + i) // bs
                block = table[r, j] if j < table.shape[1] else -1
                row = rows[block, (first + i) % bs].to(TYPES[out]) if block >= 0 else 0
                assert (got[at] == row).all()
                at += 1
