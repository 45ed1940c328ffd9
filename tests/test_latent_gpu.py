"""Absorbed attention over the latent cache on the GPU against fp64, within the
bounds of ``oracle.latent``, which follow from fp32 sums and weights in the
cache's type."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch, LatentCache  # noqa: E402
from graftrepository_amd.payload import DeviceArray  # noqa: E402
from oracle import latent as law  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(dtype) if dtype is not None else t


def host(t):
    return t.double().cpu().numpy()


class Setup:
    """Random rows, tables dealt from a shuffled pool; rows that no token sees
    hold NaN."""

    def __init__(self, ctx, new, rank, rope, bs, heads, name="bf16", seed=0, width=None, holes=(),
                 extra=0, spread=0.3, window=0, max_new=None):
        rng = np.random.default_rng(seed)
        self.rng, self.ctx, self.new, self.bs = rng, list(ctx), list(new), bs
        self.rank, self.rope, self.heads, self.name = rank, rope, heads, name
        total = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
        self.width = width if width is not None else max(total, default=0) + 1
        pool = sum(total) + 3
        ids = rng.permutation(pool).astype(np.int32)
        self.table = np.full((len(ctx), self.width), -1, np.int32)
        at = 0
        for r, t in enumerate(total):
            self.table[r, :min(t, self.width)] = ids[at:at + min(t, self.width)]
            at += t
        for r, j in holes:
            self.table[r, j] = -1
        values = rank + rope
        rows = rng.standard_normal((pool, bs, values)) * np.exp(spread * rng.standard_normal(values))
        seen = np.zeros((pool, bs), bool)
        for r, (c, n) in enumerate(zip(ctx, new)):
            for p in range(max(0, c + 1 - window) if window else 0, c + n):
                if p // bs < self.width and self.table[r, p // bs] >= 0:
                    seen[self.table[r, p // bs], p % bs] = True
        rows[~seen] = np.nan
        self.rows = dev(rows, TYPES[name])
        self.tokens = sum(new) + extra
        self.q = dev(rng.standard_normal((self.tokens, heads, values)) * 0.7, TYPES[name])
        self.scale = 1.0 / np.sqrt(values / 3)
        self.window = window
        self.max_new = max(new, default=0) if max_new is None else max_new

    def batch(self, **kw):
        b = KvBatch(dev(np.array(self.ctx, np.int32)), dev(np.array(self.new, np.int32)),
                    dev(self.table), self.bs, tokens=self.tokens, max_new=self.max_new,
                    heads=self.heads, kv_heads=1, window=self.window, latent=True, **kw)
        return b.plan()

    def check(self, out, lse, scale=None, heads_of=None, skip=()):
        rows = np.where(np.isnan(host(self.rows)), 0.0, host(self.rows))
        want, wl, ob, lb = law.attend(host(self.q), rows, self.rank, self.ctx, self.new, self.table,
                                      self.scale if scale is None else scale, self.window, self.name,
                                      heads_of)
        n = sum(self.new)
        hs = slice(None) if heads_of is None else list(heads_of)
        keep = [i for i in range(n) if i not in skip]
        off = np.abs(host(out) - want)[keep][:, hs]
        assert np.isfinite(host(out)[keep][:, hs]).all()
        worst = (off / np.maximum(ob[keep][:, hs], 1e-30)).max() if off.size else 0
        assert worst <= 1, f"output off by {worst} bounds"
        if lse is not None:
            got = host(lse)[keep][:, hs]
            none = np.isinf(wl[keep][:, hs])
            assert (got[none] == -np.inf).all()
            off = np.abs(got[~none] - wl[keep][:, hs][~none])
            assert (off <= lb[keep][:, hs][~none]).all()


SMALL = [
    # ctx, new, heads
    ([0], [1], 1), ([0], [1], 16), ([31], [1], 16), ([32], [1], 40), ([63, 0, 200], [1, 1, 1], 16),
    ([500, 17, 96], [1, 1, 1], 40), ([130, 70], [1, 1], 128), ([5, 0], [3, 2], 8),
    ([100, 0, 40], [1, 70, 3], 16), ([0, 33], [37, 1], 40), ([17], [9], 128), ([64, 1], [2, 2], 30),
    ([200, 0], [0, 4], 20), ([3, 3, 3], [0, 0, 0], 16), ([1000], [1], 5), ([7] * 40, [1] * 40, 3),
]


@pytest.mark.parametrize("ctx,new,heads", SMALL)
@pytest.mark.parametrize("rank,rope", [(512, 64), (256, 32)])
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("bs", [16, 128])
def test_attend_matches_the_law(hip_lib, ctx, new, heads, rank, rope, name, bs):
    s = Setup(ctx, new, rank, rope, bs, heads, name, extra=2)
    out = torch.full((s.tokens, heads, rank), 7.0, device="cuda", dtype=TYPES[name])
    cache = LatentCache(s.rows, rank)
    got, lse = cache.attend(s.batch(), s.q, s.scale, out=out, return_lse=True)
    assert got is out and (out[sum(new):] == 7).all()   # rows of no token stay
    s.check(out, lse, heads_of=range(0, heads, max(1, heads // 6)))


@pytest.mark.parametrize("rank,rope,heads", [(16, 16, 2), (48, 0, 3), (512, 0, 4), (128, 64, 130),
                                             (256, 64, 16), (496, 128, 1), (256, 32, 129)])
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_any_shape_of_row(hip_lib, rank, rope, heads, name):
    s = Setup([70, 0, 300], [1, 5, 2], rank, rope, 32, heads, name, extra=1, holes=[(2, 3)])
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.check(out, lse, heads_of=range(0, heads, max(1, heads // 4)))


@pytest.mark.parametrize("heads", [16, 30, 64, 128])
@pytest.mark.parametrize("rank,rope", [(512, 64), (256, 32)])
def test_long_contexts_are_cut_and_joined(hip_lib, heads, rank, rope):
    s = Setup([4000, 9, 1500], [1, 1, 1], rank, rope, 64, heads, "bf16", seed=3)
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.check(out, lse, heads_of=[0, heads // 2, heads - 1])
    again, lse2 = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("window", [1, 5, 31, 32, 100])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 3]])
@pytest.mark.parametrize("rank,rope", [(512, 64), (256, 32), (64, 16)])
def test_windows(hip_lib, window, new, rank, rope):
    s = Setup([150, 0, 63], new, rank, rope, 16, 16, "bf16", window=window)
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.check(out, lse, heads_of=[0, 7, 15])


@pytest.mark.parametrize("rank,rope", [(512, 64), (256, 32), (64, 16)])
@pytest.mark.parametrize("heads", [16, 40])
def test_missing_blocks_are_not_seen(hip_lib, rank, rope, heads):
    s = Setup([150, 40, 20], [1, 20, 1], rank, rope, 16, heads, "f16",
              holes=[(0, 2), (0, 6), (1, 0), (1, 1), (1, 2), (1, 3), (2, 0), (2, 1)], width=8)
    # (request 0's tokens from 128 on have no column of the table)
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.check(out, lse, heads_of=[0, heads - 1])
    assert torch.isinf(lse[21]).all() and (out[21] == 0).all()


def test_a_table_without_columns(hip_lib):
    s = Setup([0, 5], [1, 1], 512, 64, 16, 16, width=0)
    out, lse = LatentCache(s.rows, 512).attend(s.batch(), s.q, s.scale, return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all()


@pytest.mark.parametrize("rank,rope,heads", [(512, 64, 16), (512, 64, 40), (512, 64, 128),
                                             (256, 32, 40), (256, 32, 4), (64, 16, 4)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite_reach_only_who_sees_them(hip_lib, rank, rope, heads, bad):
    ctx, new = [90, 40], [6, 1]
    s = Setup(ctx, new, rank, rope, 32, heads, "bf16", window=0)
    # a new row of request 0 in its latent, and an old one of request 1 in its key
    s.rows[int(s.table[0, 92 // 32]), 92 % 32, 3] = bad
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.rows[int(s.table[0, 92 // 32]), 92 % 32, 3] = 0.0
    seers = range(2, 6)
    assert torch.isnan(out[2:6]).all() and torch.isnan(lse[2:6]).all()
    s.check(out, lse, heads_of=[0, heads - 1], skip=seers)
    s.rows[int(s.table[1, 1]), 5, rank + 1] = bad
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    assert torch.isnan(out[6]).all() and torch.isnan(lse[6]).all()
    s.rows[int(s.table[1, 1]), 5, rank + 1] = 0.0
    s.check(out, lse, heads_of=[0, heads - 1], skip=[6])


def test_a_window_leaves_a_bad_row_behind(hip_lib):
    s = Setup([90], [6], 512, 64, 32, 16, "bf16", window=20)
    s.rows[int(s.table[0, 2]), 73 % 32, 3] = float("inf")   # tokens 90 .. 92 see it
    out, lse = LatentCache(s.rows, 512).attend(s.batch(), s.q, s.scale, return_lse=True)
    assert torch.isnan(out[:3]).all()
    s.rows[int(s.table[0, 2]), 73 % 32, 3] = 0.0
    s.check(out, lse, skip=range(3))


def test_a_query_that_is_not_finite_stays_in_its_row(hip_lib):
    s = Setup([100, 30], [2, 1], 512, 64, 16, 16)
    s.q[1, 4, 9] = float("nan")
    out, lse = LatentCache(s.rows, 512).attend(s.batch(), s.q, s.scale, return_lse=True)
    assert torch.isnan(out[1, 4]).all() and torch.isnan(lse[1, 4])
    s.q[1, 4, 9] = 0.0
    s.check(out, lse, heads_of=[0, 3, 5, 15])


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("rank,rope", [(512, 64), (64, 16)])
def test_scales(hip_lib, scale, rank, rope):
    s = Setup([300], [3], rank, rope, 16, 16, "f16", spread=0.0)
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, scale, return_lse=True)
    s.check(out, lse, scale=scale, heads_of=[0, 9])


def test_strides_alignment_and_device_arrays(hip_lib):
    s = Setup([100, 3], [1, 2], 256, 32, 16, 8, "f16")
    cache = LatentCache(s.rows, 256)
    b = s.batch()
    want = cache.attend(b, s.q, s.scale)
    wide = torch.zeros((3, 10, 300), device="cuda", dtype=torch.float16)
    for q in (wide[:, 1:9, 8:296], wide[:, 2:, 1:289]):   # aligned rows, and not
        q.copy_(s.q)
        assert torch.equal(cache.attend(b, q, s.scale), want)
        base = torch.full((3, 9, 270), 5.0, device="cuda", dtype=torch.float16)
        out = base[:, 1:, 3:259]
        cache.attend(b, q, s.scale, out=out)
        assert torch.equal(out, want) and (base[:, 0] == 5).all() and (base[..., 259:] == 5).all()
    arrays = [DeviceArray.from_host(t.cpu().numpy()) for t in (s.rows, s.q)]
    ints = [DeviceArray.from_host(np.array(a, np.int32)) for a in (s.ctx, s.new, s.table)]
    b = KvBatch(*ints, 16, tokens=3, max_new=2, heads=8, kv_heads=1, latent=True).plan()
    got = LatentCache(arrays[0], 256).attend(b, arrays[1], s.scale)
    np.testing.assert_array_equal(got.to_host(), want.cpu().numpy())


def test_lengths_past_the_batch_are_not_written(hip_lib):
    # more tokens than rows: what fits is attended or left, nothing else is touched
    s = Setup([40, 10], [3, 30], 512, 64, 16, 16)
    b = KvBatch(dev(np.array(s.ctx, np.int32)), dev(np.array([3, 1 << 30], np.int32)), dev(s.table),
                16, tokens=20, max_new=30, heads=16, kv_heads=1, latent=True).plan()
    base = torch.full((40, 16, 512), 5.0, device="cuda", dtype=torch.bfloat16)
    LatentCache(s.rows, 512).attend(b, s.q[:20], s.scale, out=base[:20])
    assert (base[20:] == 5).all()
    s.new = [3, 0]
    s.check(base[:33], None, heads_of=[0, 8])


@pytest.mark.parametrize("rank,heads", [(512, 16), (256, 40), (64, 4)])
def test_a_captured_step_follows_its_lengths(hip_lib, rank, heads):
    rope = {512: 64, 256: 32, 64: 16}[rank]
    s = Setup([100, 37], [1, 1], rank, rope, 16, heads, width=20)
    ctx, new = dev(np.array(s.ctx, np.int32)), dev(np.array(s.new, np.int32))
    rows = s.rows.nan_to_num(0.25)
    table = dev(np.arange(40, dtype=np.int32).reshape(2, 20))
    rows = torch.cat([rows] * 4)[:40].contiguous()
    b = KvBatch(ctx, new, table, 16, tokens=2, max_new=1, heads=heads, kv_heads=1, latent=True)
    cache = LatentCache(rows, rank)
    out = torch.empty((2, heads, rank), device="cuda", dtype=torch.bfloat16)
    b.plan()
    cache.attend(b, s.q, s.scale, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.plan()
        cache.attend(b, s.q, s.scale, out=out)
    for step in range(3):
        ctx += 61
        graph.replay()
        torch.cuda.synchronize()
        eager = KvBatch(ctx, new, table, 16, tokens=2, max_new=1, heads=heads, kv_heads=1,
                        latent=True).plan()
        assert torch.equal(cache.attend(eager, s.q, s.scale), out)


def test_two_streams_with_a_batch_each(hip_lib):
    s = Setup([700, 300], [1, 1], 512, 64, 16, 16)
    cache = LatentCache(s.rows, 512)
    want = cache.attend(s.batch(), s.q, s.scale)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            b = s.batch()
            got.append([cache.attend(b, s.q, s.scale) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for gs in got for g in gs)
