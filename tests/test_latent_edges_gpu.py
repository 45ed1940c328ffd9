"""What the latent operators' callers do besides one plain call: streams, graphs,
arrays without torch, cut pieces, scales and batches without tokens."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch, KvCache, LatentCache, Rotary, attend_rows  # noqa: E402
from graftrepository_amd.payload import DeviceArray  # noqa: E402
from tests.test_latent_gpu import Setup, dev, host  # noqa: E402
from tests.test_latent_rows_gpu import Rows, ints  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64), (24, 40)])
def test_scales_over_rows(hip_lib, scale, dk, dv):
    s = Rows([150, 0], [40, 70], dk, dv, 2, "f16")
    s.scale = scale
    s.check(*s.run(softmax_scale=scale))


@pytest.mark.parametrize("dk,dv,name", [(192, 128, "bf16"), (96, 64, "f16"), (128, 128, "f16")])
@pytest.mark.parametrize("window", [0, 1500])
def test_long_rows_are_cut_and_joined(hip_lib, dk, dv, name, window):
    # few tokens and heads, so that a unit goes to many blocks
    s = Rows([4000, 700], [130, 20], dk, dv, 2, name, window=window)
    out, lse = s.run()
    s.check(out, lse, heads_of=[1])
    again, lse2 = s.run()
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64)])
@pytest.mark.parametrize("which,bad", [("v", float("inf")), ("k", float("-inf")), ("k", float("nan"))])
def test_a_bad_row_in_a_cut_unit(hip_lib, dk, dv, which, bad):
    # row 4090 is in the last of a unit's pieces, and seen by the tokens from 90 on
    s = Rows([4000], [130], dk, dv, 2, "bf16")
    getattr(s, which)[4090, 1, 5] = bad
    out, lse = s.run()
    seers = list(range(90, 130))
    assert not torch.isfinite(out[seers, 1, 5]).any()
    s.check(out, lse, skip=seers, heads_of=[1])
    s.check(out, lse, heads_of=[0])


def test_rows_on_another_stream_and_without_torch(hip_lib):
    s = Rows([60, 0], [5, 90], 96, 64, 3, "f16")
    want, wl = s.run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    b = s.batch()
    torch.cuda.synchronize()
    out, lse = attend_rows(b, s.q, s.k, s.v, ints(s.cu), return_lse=True, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wl)
    a = [DeviceArray.from_host(x.cpu().numpy()) for x in (s.q, s.k, s.v)]
    i = [DeviceArray.from_host(np.array(x, np.int32)) for x in (s.ctx, s.new, s.cu)]
    b = KvBatch(i[0], i[1], DeviceArray.from_host(np.zeros((2, 1), np.int32)), 64, tokens=s.tokens,
                max_new=90, heads=3, kv_heads=1, latent=True).plan()
    got, lse = attend_rows(b, *a, i[2], return_lse=True)
    np.testing.assert_array_equal(got.to_host(), want.cpu().numpy())
    np.testing.assert_array_equal(lse.to_host(), wl.cpu().numpy())


def test_latents_without_torch(hip_lib):
    rng = np.random.default_rng(3)
    latent, part = (rng.standard_normal((7, n)).astype(np.float32) for n in (64, 32))
    table = np.array([[2], [0]], np.int32)
    lens = [np.array(x, np.int32) for x in ([3, 0], [5, 2])]
    rotary = Rotary(32)

    def run(put, cache):
        b = KvBatch(put(lens[0]), put(lens[1]), put(table), 16, tokens=7, max_new=5, heads=2,
                    kv_heads=1, latent=True).plan()
        cache.append(b, put(latent), put(part), rotary=rotary)
        return cache.read(put(table), put(np.array([3, 0], np.int32)), put(np.array([0, 5, 7], np.int32)),
                          7, dtype="f32")

    mine = run(DeviceArray.from_host, LatentCache.empty(3, 16, 64, 32, "bf16")).to_host()
    rows = torch.zeros((3, 16, 96), device="cuda", dtype=torch.bfloat16)
    theirs = run(dev, LatentCache(rows, 64)).cpu().numpy()
    np.testing.assert_array_equal(mine, theirs)
    assert np.isfinite(mine).all()


def test_batches_without_tokens(hip_lib):
    none = torch.zeros((0, 2, 192), device="cuda", dtype=torch.bfloat16)
    rows = torch.zeros((4, 16, 288), device="cuda", dtype=torch.bfloat16)
    cache = LatentCache(rows, 256)
    for lens in ([0, 0], []):
        table = torch.zeros((len(lens), 2), device="cuda", dtype=torch.int32)
        b = KvBatch(ints(lens), ints(lens), table, 16, tokens=0, max_new=0, heads=2, kv_heads=1,
                    latent=True).plan()
        cache.append(b, rows[0, :0, :256], rows[0, :0, 256:], rotary=Rotary(32))
        assert cache.attend(b, none[..., :1].expand(0, 2, 288).contiguous(), 1.0).shape == (0, 2, 256)
        cu = ints([0] * (len(lens) + 1))
        out, lse = attend_rows(b, none, none, none[..., :128].contiguous(), cu, return_lse=True)
        assert out.shape == (0, 2, 128) and lse.shape == (0, 2)
        assert cache.read(table, ints(lens), cu, 0).shape == (0, 288)
    assert (rows == 0).all()


def test_tokens_without_rows_see_nothing(hip_lib):
    s = Rows([0, 40], [3, 50], 192, 128, 2, count=[0, 90])
    out, lse = s.run()
    assert (out[:3] == 0).all() and (lse[:3] == -float("inf")).all()
    s.check(out, lse)


@pytest.mark.parametrize("start", [-7, 1 << 30, -(1 << 30)])
def test_starts_far_from_the_tokens(hip_lib, start):
    # rows before position 0 are seen by all, rows after every token by none
    s = Rows([40, 40], [30, 30], 192, 128, 2, starts=[start, 0], count=[50, 70])
    out, lse = s.run()
    assert torch.isfinite(out).all()
    if start > 0:
        assert (out[:30] == 0).all() and (lse[:30] == -float("inf")).all()
    elif start < -1000:
        q, k, v = (host(x) for x in (s.q[:30], s.k[:50], s.v[:50]))
        for h in range(2):
            p = np.exp(s.scale * q[:, h] @ k[:, h].T)
            want = p @ v[:, h] / p.sum(1, keepdims=True)
            # weights and results round to bf16 (2^-8 each)
            bound = 2.0 ** -8 * (p @ np.abs(v[:, h]) / p.sum(1, keepdims=True) + np.abs(want)) * 1.01 + 1e-5
            assert (np.abs(host(out[:30, h]) - want) <= bound).all()


def test_a_captured_step_of_the_whole_path(hip_lib):
    """Append with a rotation, rotate the queries, attend: one graph, replayed over
    growing lengths, against the same calls one by one."""
    torch.manual_seed(5)
    sessions, rank, rope, heads, bs = 3, 256, 32, 16, 16
    rotary, k8 = Rotary(rope, layout="interleaved"), Rotary(64)
    table = torch.randperm(60, device="cuda").int().view(3, 20)
    x = dict(latent=torch.empty(sessions, rank, device="cuda"), part=torch.empty(sessions, rope, device="cuda"),
             q=torch.empty(sessions, heads, rank + rope, device="cuda", dtype=torch.bfloat16),
             k=torch.empty(sessions, 2, 64, device="cuda"), v=torch.empty(sessions, 2, 64, device="cuda"))

    def make():
        ctx = ints([0, 48, 16])  # at the beginning of blocks
        b = KvBatch(ctx, ints([1] * 3), table, bs, tokens=3, max_new=1, heads=heads, kv_heads=1, latent=True)
        rows = torch.zeros(60, bs, rank + rope, device="cuda", dtype=torch.bfloat16)
        b8 = KvBatch(ctx, ints([1] * 3), table, bs, tokens=3, max_new=1, heads=4, kv_heads=2)
        kv = KvCache.empty(60, bs, 2, 64)
        starts, cu = ints([0] * 3), ints([0, 320, 640, 960])
        back = []

        def step():
            b.plan()
            b8.plan()
            cache.append(b, x["latent"], x["part"], rotary=rotary)
            q = rotary.apply(x["q"], b.positions, start=rank)
            out = cache.attend(b, q, 0.1)
            kv.append(b8, x["k"], x["v"], rotary=k8)
            back[:] = [out, rows, b.positions]
            return back

        cache = LatentCache(rows, rank)
        return ctx, step, kv, (table, starts, cu)

    def fill(seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        for t in x.values():
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))

    ctx, step, kv, read = make()
    ctx2, step2, kv2, _ = make()
    fill(0)
    step()
    step2()                       # both have done the first step
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    captured = list(captured)
    for n in range(4):
        ctx += 1
        ctx2 += 1
        fill(n + 1)
        graph.replay()
        torch.cuda.synchronize()
        want = step2()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        table, starts, cu = read
        lens = (ctx + 1).tolist()
        cu = ints(np.concatenate([[0], np.cumsum(lens)]))
        for a, b in zip(kv.read(table, starts, cu, sum(lens), dtype="f32"),
                        kv2.read(table, starts, cu, sum(lens), dtype="f32")):
            assert torch.equal(a[:lens[0]], b[:lens[0]])  # session 0's are all written


def test_one_batch_serves_caches_of_both_widths(hip_lib):
    a = Setup([90, 3], [2, 1], 512, 64, 16, 16)
    b = Setup([90, 3], [2, 1], 256, 32, 16, 16)
    b.table = a.table
    batch = a.batch()
    big, small = LatentCache(a.rows, 512), LatentCache(b.rows.nan_to_num(0.5)[:a.rows.shape[0]], 256)
    first = [c.attend(batch, s.q, s.scale) for c, s in ((big, a), (small, b))]
    again = [c.attend(batch, s.q, s.scale) for c, s in ((big, a), (small, b))]
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    a.check(first[0], None, heads_of=[3])


def test_values_that_require_gradients_are_refused(hip_lib):
    s = Rows([0], [3], 192, 128, 2)
    for which in ("q", "k", "v"):
        x = {n: getattr(s, n) for n in ("q", "k", "v")}
        x[which] = x[which].clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            attend_rows(s.batch(), x["q"], x["k"], x["v"], ints(s.cu))
        with torch.no_grad():
            attend_rows(s.batch(), x["q"], x["k"], x["v"], ints(s.cu))
    with pytest.raises(ValueError, match="bf16 or f16"):
        attend_rows(s.batch(), s.q.float(), s.k.float(), s.v.float(), ints(s.cu))


def test_one_batch_serves_rows_of_unlike_key_parts(hip_lib):
    # of one rank, but with and without the matrix cores' kernel and its scratch
    a = Setup([600, 3], [2, 1], 512, 64, 16, 16)
    b = Setup([600, 3], [2, 1], 512, 0, 16, 16)
    b.table = a.table
    batch = a.batch()
    rows = b.rows.nan_to_num(0.5)[:a.rows.shape[0]].contiguous()
    plain = LatentCache(rows, 512).attend(batch, b.q, b.scale)
    out = LatentCache(a.rows, 512).attend(batch, a.q, a.scale)
    a.check(out, None, heads_of=[3])
    assert torch.equal(LatentCache(rows, 512).attend(batch, b.q, b.scale), plain)


def test_more_requests_than_the_plan_holds_in_lds(hip_lib):
    n, heads = 5000, 4
    rng = np.random.default_rng(9)
    ctx = rng.integers(0, 15, n)
    table = dev(rng.permutation(n).astype(np.int32)[:, None])
    rows = dev(rng.standard_normal((n, 16, 288)), torch.bfloat16)
    q = dev(rng.standard_normal((n, heads, 288)), torch.bfloat16)
    k = dev(rng.standard_normal((n, heads, 96)), torch.bfloat16)
    v = dev(rng.standard_normal((n, heads, 64)), torch.bfloat16)
    cache = LatentCache(rows, 256)

    def run(a, b):
        batch = KvBatch(ints(ctx[a:b]), ints([1] * (b - a)), table[a:b], 16, tokens=b - a, max_new=1,
                        heads=heads, kv_heads=1, latent=True).plan()
        cu = ints(np.arange(b - a + 1))
        return (cache.attend(batch, q[a:b], 0.1),
                attend_rows(batch, k[a:b], k[a:b], v[a:b], cu, starts=ints(ctx[a:b])))

    # a tile to a request: nothing is cut, and every request's result its own
    whole, halves = run(0, n), [run(0, 2500), run(2500, n)]
    for i in range(2):
        assert torch.equal(whole[i], torch.cat([h[i] for h in halves]))
    assert torch.equal(whole[1], v)           # of one row that a token sees


def test_rows_past_4_gib_of_a_cache(hip_lib):
    blocks, bs, rank, rope, heads = 59000, 64, 512, 64, 16
    big = torch.empty((blocks, bs, rank + rope), device="cuda", dtype=torch.bfloat16)
    small = torch.zeros((4, bs, rank + rope), device="cuda", dtype=torch.bfloat16)
    assert big.numel() * 2 > 1 << 32
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randn(200, rank + rope, generator=gen, device="cuda")
    q = torch.randn(1, heads, rank + rope, generator=gen, device="cuda").bfloat16()
    w = (torch.randn(heads, 256, rank, generator=gen, device="cuda") / rank ** 0.5).bfloat16()
    rotary, got = Rotary(rope), []
    for rows, ids in ((big, [blocks - 1, 3, blocks - 2, blocks - 3]), (small, [0, 1, 2, 3])):
        table = ints([ids])
        cache = LatentCache(rows, rank)
        b = KvBatch(ints([0]), ints([200]), table, bs, tokens=200, max_new=200, heads=heads, kv_heads=1,
                    latent=True).plan()
        cache.append(b, x[:, :rank], x[:, rank:], rotary=rotary)
        one = KvBatch(ints([199]), ints([1]), table, bs, tokens=1, max_new=1, heads=heads, kv_heads=1,
                      latent=True).plan()
        cu = ints([0, 200])
        got.append([cache.attend(one, q, 0.05), cache.read(table, ints([0]), cu, 200),
                    *cache.expand(w, 128, table, ints([0]), cu, 200)])
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_dense_rows_past_4_gib(hip_lib):
    s = Rows([100], [40], 192, 128, 2, "bf16")
    want, lse = s.run()
    n, stride = 140, 1 << 24                 # 32 MiB from row to row
    base = torch.empty(n * stride, device="cuda", dtype=torch.bfloat16)
    for name, d in (("k", 192), ("v", 128)):
        far = base.as_strided((n, 2, d), (stride, d, 1), 0 if name == "k" else 1024)
        far.copy_(getattr(s, name))
        setattr(s, name, far)
    out, lse2 = s.run()
    assert torch.equal(out, want) and torch.equal(lse, lse2)


def test_two_streams_over_rows_with_a_batch_each(hip_lib):
    s = Rows([3000, 40], [60, 200], 96, 64, 4, "f16")
    want, _ = s.run()
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(st):
            b = s.batch()
            got += [attend_rows(b, s.q, s.k, s.v, ints(s.cu), starts=ints(s.starts)) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_heads_that_share_rows(hip_lib):
    # strides of 0: every head has the same keys and values
    s = Rows([50, 0], [30, 80], 128, 128, 3, "bf16")
    k, v = s.k[:, :1].clone(), s.v[:, :1].clone()
    s.k, s.v = k.expand(-1, 3, -1).contiguous(), v.expand(-1, 3, -1).contiguous()
    want, _ = s.run()
    s.k, s.v = k.expand(-1, 3, -1), v.expand(-1, 3, -1)
    got, _ = s.run()
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [130, 250, 300, 1100])
@pytest.mark.parametrize("rank,rope,heads", [(512, 64, 128), (256, 32, 40)])
def test_fewer_and_more_sessions_than_runs(hip_lib, n, rank, rope, heads):
    # runs of a session's own, runs that go on from one to the next, and lists longer than
    # a block plans at once
    rng = np.random.default_rng(n)
    ctx = rng.integers(0, 300 if n < 1000 else 90, n).tolist()
    s = Setup(ctx, [1] * n, rank, rope, 32, heads, "f16")
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.check(out, lse, heads_of=[heads - 1])
