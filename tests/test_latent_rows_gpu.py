"""The expanded form of latent attention on the GPU against fp64, within the
bounds of ``oracle.latent``."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch, LatentCache, attend_rows  # noqa: E402
from oracle import latent as law  # noqa: E402
from tests.test_latent_gpu import TYPES, Setup, dev, host  # noqa: E402

pytestmark = pytest.mark.gpu


def ints(a):
    return dev(np.array(a, np.int32))


EXPANDS = [
    # rank, rope, heads, key, value
    (512, 64, 3, 128, 128), (256, 32, 5, 64, 64), (32, 16, 1, 8, 16), (64, 0, 7, 40, 24),
    (48, 32, 4, 32, 16), (512, 64, 2, 192, 256), (96, 16, 40, 16, 8),
]


@pytest.mark.parametrize("rank,rope,heads,key,value", EXPANDS)
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_expand_matches_the_law(hip_lib, rank, rope, heads, key, value, name):
    s = Setup([150, 3, 40], [1, 1, 1], rank, rope, 16, 1, name, holes=[(0, 2)])
    s.rows.nan_to_num_(0.5)
    cache = LatentCache(s.rows, rank)
    weight = dev(s.rng.standard_normal((heads, key + value, rank)) / np.sqrt(rank), TYPES[name])
    starts, count = [5, 0, 38], [140, 4, 60]      # the last goes past its blocks
    cu = np.concatenate([[0], np.cumsum(count)])
    k, v = cache.expand(weight, key, ints(s.table), ints(starts), ints(cu), int(cu[-1]))
    assert k.shape == (204, heads, key + rope) and v.shape == (204, heads, value)
    wk, wv, kb, vb = law.expand(host(s.rows), host(weight), key, rank,
                                list(zip(range(3), starts, count)), s.table, name)
    assert (np.abs(host(k) - wk) <= kb).all() and (np.abs(host(v) - wv) <= vb).all()
    none = cache.expand(weight, key, ints(s.table), ints(starts), ints([0, 0, 0, 0]), 0)
    assert none[0].shape == (0, heads, key + rope)


def test_rows_that_are_not_finite_expand_to_themselves_only(hip_lib):
    s = Setup([60], [1], 512, 64, 16, 1)
    s.rows.nan_to_num_(0.5)
    cache = LatentCache(s.rows, 512)
    weight = dev(s.rng.standard_normal((2, 256, 512)), torch.bfloat16)
    args = (ints(s.table), ints([0]), ints([0, 61]), 61)
    k, v = cache.expand(weight, 128, *args)
    s.rows[int(s.table[0, 1]), 4, 100] = float("nan")
    k2, v2 = cache.expand(weight, 128, *args)
    assert torch.isnan(k2[20, :, :128]).all() and torch.isnan(v2[20]).all()
    keep = [i for i in range(61) if i != 20]
    assert torch.equal(k2[keep], k[keep]) and torch.equal(v2[keep], v[keep])
    assert torch.equal(k2[20, :, 128:], k[20, :, 128:])


class Rows:
    """Dense rows of requests and the queries of a batch over them."""

    def __init__(self, ctx, new, dk, dv, heads, name="bf16", window=0, starts=None, count=None,
                 extra=0, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.new, self.heads, self.name, self.window = ctx, new, heads, name, window
        self.starts = [0] * len(ctx) if starts is None else starts
        count = [c + n - a for c, n, a in zip(ctx, new, self.starts)] if count is None else count
        self.cu = np.concatenate([[0], np.cumsum(count)])
        n, t = int(self.cu[-1]), sum(new) + extra
        self.k = dev(rng.standard_normal((n, heads, dk)), TYPES[name])
        self.v = dev(rng.standard_normal((n, heads, dv)), TYPES[name])
        self.q = dev(rng.standard_normal((t, heads, dk)), TYPES[name])
        self.tokens, self.scale = t, 1.0 / np.sqrt(dk)

    def batch(self):
        return KvBatch(ints(self.ctx), ints(self.new), torch.zeros((len(self.ctx), 1), dtype=torch.int32,
                       device="cuda"), 64, tokens=self.tokens, max_new=max(self.new),
                       heads=self.heads, kv_heads=1, window=self.window, latent=True).plan()

    def run(self, **kw):
        return attend_rows(self.batch(), self.q, self.k, self.v, ints(self.cu),
                           starts=ints(self.starts), return_lse=True, **kw)

    def check(self, out, lse, heads_of=None, skip=()):
        k, v = (np.nan_to_num(host(x), nan=0.0, posinf=0.0, neginf=0.0) for x in (self.k, self.v))
        want, wl, ob, lb = law.attend_rows(host(self.q), k, v, self.ctx, self.new, self.cu, self.starts,
                                           self.scale, self.window, self.name, heads_of)
        hs = slice(None) if heads_of is None else list(heads_of)
        keep = [i for i in range(sum(self.new)) if i not in skip]
        assert np.isfinite(host(out)[keep][:, hs]).all()
        off = np.abs(host(out) - want)[keep][:, hs]
        assert (off <= ob[keep][:, hs]).all(), (off / np.maximum(ob[keep][:, hs], 1e-30)).max()
        got, wl, lb = host(lse)[keep][:, hs], wl[keep][:, hs], lb[keep][:, hs]
        none = np.isinf(wl)
        assert (got[none] == -np.inf).all()
        assert (np.abs(got[~none] - wl[~none]) <= lb[~none]).all()


DIMS = [(192, 128), (96, 64), (128, 128), (64, 64), (40, 200), (8, 8), (512, 16)]


@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0, 0, 7], [33, 130, 1]), ([100, 5], [129, 300]),
                                     ([31, 0], [1, 32]), ([260], [64])])
def test_attend_rows_matches_the_law(hip_lib, dk, dv, name, ctx, new):
    s = Rows(ctx, new, dk, dv, 3, name, extra=2)
    out = torch.full((s.tokens, 3, dv), 7.0, device="cuda", dtype=TYPES[name])
    got, lse = s.run(out=out)
    assert got is out and (out[sum(new):] == 7).all()
    s.check(out, lse, heads_of=[0, 2])


@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64), (24, 40)])
@pytest.mark.parametrize("window", [1, 20, 64, 150])
def test_windows_over_rows(hip_lib, dk, dv, window):
    s = Rows([90, 0], [200, 40], dk, dv, 2, window=window)
    s.check(*s.run())


@pytest.mark.parametrize("dk,dv", [(192, 128), (128, 128), (24, 40)])
def test_parts_of_rows_join_by_their_statistics(hip_lib, dk, dv):
    whole = Rows([300], [70], dk, dv, 2, "f16")
    out, lse = whole.run()
    parts = []
    for a, b in ((0, 130), (130, 310), (310, 370)):
        p = Rows([300], [70], dk, dv, 2, "f16", starts=[a], count=[b - a])
        p.q, p.k, p.v = whole.q, whole.k[a:b].contiguous(), whole.v[a:b].contiguous()
        o, e = p.run()
        p.check(o, e)
        parts.append((o.double(), e.double()))
    top = torch.stack([e for _, e in parts]).amax(0)
    w = [torch.exp(e - top) for _, e in parts]
    joined = sum(o * x[..., None] for (o, _), x in zip(parts, w)) / sum(w)[..., None]
    # each part and the whole round to fp16 (half a step) and round weights so
    bound = 4 * 2.0 ** -11 * sum(o.abs() * x[..., None] for (o, _), x in zip(parts, w)) / sum(w)[..., None]
    assert ((joined - out.double()).abs() <= bound + 2.0 ** -9).all()
    assert (torch.isinf(parts[2][1][:9])).all()       # tokens before that part's first row


@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64), (24, 40)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("window", [0, 50])
def test_bad_rows_reach_only_who_sees_them(hip_lib, dk, dv, bad, which, window):
    s = Rows([60, 10], [140, 30], dk, dv, 2, window=window)
    # a row of request 0 that its tokens from 90 on see (in a window, 90 .. 139)
    getattr(s, which)[90, 1, 3] = bad
    out, lse = s.run()
    seers = [i for i in range(140) if 60 + i >= 90 and (not window or 60 + i < 90 + window)]
    assert not torch.isfinite(out[seers, 1, 3]).any()
    s.check(out, lse, skip=seers, heads_of=[1])
    s.check(out, lse, heads_of=[0])


def test_rows_of_any_strides(hip_lib):
    s = Rows([20], [40], 192, 128, 3, "f16")
    want, _ = s.run()
    for at in (8, 1):
        wide = [torch.zeros((n, 4, d + 16), device="cuda", dtype=torch.float16)
                for n, d in ((40, 192), (60, 192), (60, 128))]
        q, k, v = (w[:, 1:, at:at + x.shape[2]] for w, x in zip(wide, (s.q, s.k, s.v)))
        for to, x in ((q, s.q), (k, s.k), (v, s.v)):
            to.copy_(x)
        base = torch.full((40, 4, 144), 3.0, device="cuda", dtype=torch.float16)
        out = base[:, :3, at:at + 128]
        attend_rows(s.batch(), q, k, v, ints(s.cu), out=out)
        assert torch.equal(out, want) and (base[:, 3] == 3).all() and (base[..., :at] == 3).all()


@pytest.mark.parametrize("rank,rope,heads,key,value", [(512, 64, 4, 128, 128), (256, 32, 6, 64, 64)])
def test_the_two_forms_agree(hip_lib, rank, rope, heads, key, value):
    """Absorbed queries and outputs through the weights are the expanded form's,
    by fp64 arithmetic on the kernels' own inputs and outputs."""
    s = Setup([70, 0], [40, 33], rank, rope, 32, heads, "f16", spread=0.0)
    s.rows.nan_to_num_(0.0)
    cache = LatentCache(s.rows, rank)
    w = dev(s.rng.standard_normal((heads, key + value, rank)) / np.sqrt(rank), torch.float16)
    q = dev(s.rng.standard_normal((s.tokens, heads, key + rope)), torch.float16)
    scale = 1.0 / np.sqrt(key + rope)
    cu = ints([0, 110, 143])
    b = s.batch()
    k, v = cache.expand(w, key, ints(s.table), ints([0, 0]), cu, 143)
    out = attend_rows(b, q, k, v, cu, softmax_scale=scale)
    wk, wv = w[:, :key].double(), w[:, key:].double()
    absorbed = torch.cat([torch.matmul(q[..., :key].double().transpose(0, 1), wk).transpose(0, 1),
                          q[..., key:].double()], -1).half()
    o = cache.attend(b, absorbed.contiguous(), scale).double()
    o = torch.matmul(o.transpose(0, 1), wv.transpose(1, 2).contiguous()).transpose(0, 1)
    # fp16 roundings of k, v, weights and outputs in one form, of q, weights and the
    # mean latent in the other: half steps 2^-11 each.  A score of size S is off by
    # 2^-11 times its terms' 2-norm (about S's own scale, 1) in each form, which
    # moves a mean of values of size 1 by as much; the mean latent's rounding
    # comes back through `rank` terms of size 1/sqrt(rank).  16 such in all, and the
    # largest of 70000 normal deviates (5) of each.
    assert (out.double() - o).abs().max() <= 16 * 5 * 2.0 ** -11


def test_a_captured_prompt_follows_its_lengths(hip_lib):
    s = Rows([0, 50], [100, 60], 192, 128, 2)
    ctx, new, cu = ints(s.ctx), ints(s.new), ints(s.cu)
    table = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    make = lambda: KvBatch(ctx, new, table, 64, tokens=160, max_new=100, heads=2, kv_heads=1,  # noqa: E731
                           latent=True)
    b = make()
    out = torch.zeros_like(s.q[..., :128])
    b.plan()
    attend_rows(b, s.q, s.k, s.v, cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.plan()
        attend_rows(b, s.q, s.k, s.v, cu, out=out)
    for step in range(3):
        new.copy_(ints([90 - 20 * step, 70 + 20 * step]))
        ctx.copy_(ints([10 + 20 * step, 40 - 20 * step]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(attend_rows(make().plan(), s.q, s.k, s.v, cu), out)
