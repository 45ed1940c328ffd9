"""The 8-bit key/value cache on the GPU against its laws on the host.

Block tables, slot maps, codes, scales and values read back are compared bit
for bit (whole numbers, and single fp32 operations).  Attention is compared
with fp64 within ``oracle.kv.attend``'s bound, which follows from fp32 sums
and fp16 probabilities.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch, KvCache  # noqa: E402
from graftrepository_amd.payload import DeviceArray  # noqa: E402
from oracle import kv as law  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(dtype) if dtype is not None else t


def lens(*pairs):
    return [p[0] for p in pairs], [p[1] for p in pairs]


class Setup:
    """Random cache, tables dealt from a shuffled pool; blocks of nobody hold
    NaN scales, and places past a request's end hold any codes."""

    def __init__(self, ctx, new, kv, hd, bs, seed=0, spare=3, width=None, holes=(), extra_rows=0):
        rng = np.random.default_rng(seed)
        self.rng, self.ctx, self.new, self.bs = rng, list(ctx), list(new), bs
        total = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
        self.width = width if width is not None else max(total, default=0) + 1
        pool = sum(total) + spare
        ids = rng.permutation(pool).astype(np.int32)
        self.table = np.full((len(ctx), self.width), -1, np.int32)
        at = 0
        for r, t in enumerate(total):
            t = min(t, self.width)
            self.table[r, :t] = ids[at:at + t]
            at += t
        for r, j in holes:
            self.table[r, j] = -1
        shape = (pool, kv, bs, hd)
        self.kc = np.clip(np.rint(rng.standard_normal(shape) * 33), -127, 127).astype(np.int8)
        self.vc = np.clip(np.rint(rng.standard_normal((pool, kv, hd, bs)) * 33), -127,
                          127).astype(np.int8)
        self.ks = (np.exp(0.5 * rng.standard_normal((pool, kv))) / 36).astype(np.float32)
        self.vs = (np.exp(0.5 * rng.standard_normal((pool, kv))) / 36).astype(np.float32)
        nobody = np.setdiff1d(np.arange(pool), self.table[self.table >= 0])
        self.ks[nobody] = np.nan
        self.vs[nobody] = np.nan
        self.kv, self.hd = kv, hd
        self.tokens = sum(new) + extra_rows

    def cache(self):
        return KvCache(dev(self.kc), dev(self.vc), dev(self.ks), dev(self.vs))

    def batch(self, heads=None, window=0, **kw):
        b = KvBatch(dev(np.array(self.ctx, np.int32)), dev(np.array(self.new, np.int32)),
                    dev(self.table), self.bs, tokens=self.tokens,
                    max_new=max(self.new, default=0), heads=heads or self.kv, kv_heads=self.kv,
                    window=window, **kw)
        return b.plan()


# -------------------------------------------------------------------- plan

PLANS = [
    ([0], [1], 16),
    ([15, 16, 17, 0], [1, 1, 1, 0], 16),
    ([0, 0, 0], [0, 0, 0], 32),
    ([31, 64, 0, 100, 7], [33, 64, 1, 0, 300], 32),
    (list(range(0, 1200)), [1] * 1200, 64),
    ([5] * 5000, [(i * 7) % 4 for i in range(5000)], 16),
    ([0, 3], [9000, 9001], 128),
]


@pytest.mark.parametrize("ctx,new,bs", PLANS)
@pytest.mark.parametrize("short", [False, True])
def test_plan_matches_the_law(hip_lib, ctx, new, bs, short):
    rng = np.random.default_rng(len(ctx))
    held = [-(-c // bs) for c in ctx]
    need = sum(max(0, -(-(c + n) // bs) - h) if n else 0 for c, n, h in zip(ctx, new, held))
    width = max(-(-(c + n) // bs) for c, n in zip(ctx, new))
    width = max(1, width - (1 if short else 0))     # a table too narrow for the longest
    ids = rng.permutation(sum(held) + need + 5).astype(np.int32)
    table = np.full((len(ctx), width), -7, np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :min(h, width)] = ids[at:at + min(h, width)]
        at += h
    free = ids[at:at + (need * 2 // 3 if short else need + 2)]
    tokens = sum(new) + 3
    head = dev(np.array([0], np.int32))
    b = KvBatch(dev(np.array(ctx, np.int32)), dev(np.array(new, np.int32)), dev(table), bs,
                tokens=tokens, max_new=max(new), heads=4, kv_heads=2, free_list=dev(free),
                free_head=head)
    want = law.plan(ctx, new, table, bs, tokens, list(free), 0)
    for _ in range(2):                              # the same again: nothing is used up
        b.plan()
        got = (b.block_table, b.cu_new, b.slot_map, b.positions)
        for g, w in zip(got, want[:4]):
            np.testing.assert_array_equal(g.cpu().numpy(), w)
        assert int(b.free_head_out) == want[4]


def test_plan_goes_on_where_the_last_one_ended(hip_lib):
    bs, steps = 16, 40
    ctx = np.array([0, 14, 31], np.int32)
    table = np.full((3, 8), -1, np.int32)
    table[1, 0], table[2, :2] = 90, (91, 92)
    free = np.arange(10, 60, dtype=np.int32)
    d_ctx, d_table = dev(ctx), dev(table)
    b = KvBatch(d_ctx, dev(np.ones(3, np.int32)), d_table, bs, tokens=3, max_new=1, heads=2,
                kv_heads=2, free_list=dev(free), free_head=dev(np.zeros(1, np.int32)))
    head = 0
    for _ in range(steps):
        b.plan()
        table, _, slots, _, head = law.plan(ctx.tolist(), [1, 1, 1], table, bs, 3, list(free), head)
        np.testing.assert_array_equal(b.slot_map.cpu().numpy(), slots)
        b.advance()
        d_ctx += 1
        ctx = ctx + 1
    np.testing.assert_array_equal(d_table.cpu().numpy(), table)
    assert int(b.free_head) == head


# ---------------------------------------------------------- append and read

APPENDS = [
    # ctx, new, kv, hd, block
    ([0], [1], 1, 16, 16),
    ([3, 16, 0, 40], [1, 1, 1, 0], 2, 128, 16),
    ([0, 5, 33, 64], [40, 64, 1, 100], 3, 64, 32),
    ([17, 0], [300, 129], 4, 256, 64),
    ([100, 127, 128], [1, 2, 130], 2, 80, 128),
    ([9] * 70, [1] * 70, 8, 128, 64),
]


@pytest.mark.parametrize("ctx,new,kv,hd,bs", APPENDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("strided", [False, True])
def test_append_and_read_match_the_law(hip_lib, ctx, new, kv, hd, bs, dtype, strided):
    s = Setup(ctx, new, kv, hd, bs, seed=hd + bs)
    # louder and softer than what a block holds: scales that grow and stay
    loud = np.exp(s.rng.standard_normal((s.tokens, 1, 1)) * 1.2)
    x = [(s.rng.standard_normal((s.tokens, kv, hd)) * loud).astype(np.float32) for _ in "kv"]
    t = [dev(a, TYPES[dtype]) for a in x]
    x = [a.float().cpu().numpy() for a in t]
    if strided:   # rows inside a wider projection, heads padded
        wide = torch.zeros(s.tokens, kv, 2 * hd + 8, dtype=TYPES[dtype], device="cuda")
        wide[:, :, 1:1 + hd] = t[0]
        wide[:, :, 1 + hd:1 + 2 * hd] = t[1]
        t = [wide[:, :, 1:1 + hd], wide[:, :, 1 + hd:1 + 2 * hd]]
    cache, batch = s.cache(), s.batch()
    for _ in range(2):                              # a step done again changes nothing
        cache.append(batch, *t)
        law.append(s.kc, s.ks, x[0], ctx, new, s.table, False)
        law.append(s.vc, s.vs, x[1], ctx, new, s.table, True)
        np.testing.assert_array_equal(cache.k_scales.cpu().numpy(), s.ks)
        np.testing.assert_array_equal(cache.v_scales.cpu().numpy(), s.vs)
        np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)
        np.testing.assert_array_equal(cache.v_codes.cpu().numpy(), s.vc)
    # read back from odd places, one request not at all
    starts = np.array([c // 3 for c in ctx], np.int32)
    count = [c + n - st for c, n, st in zip(ctx, new, starts)]
    count[0] = min(count[0], 1)
    cu = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    for out in ("f32", "bf16", "f16"):
        k, v = cache.read(dev(s.table), dev(starts), dev(cu), int(cu[-1]), dtype=out)
        for got, codes, scales, tr in ((k, s.kc, s.ks, False), (v, s.vc, s.vs, True)):
            want = [law.values(codes, scales, s.table[r], tr)[starts[r]:starts[r] + count[r]]
                    for r in range(len(ctx))]
            want = torch.from_numpy(np.concatenate(want)).to(TYPES[out])
            assert torch.equal(got.cpu(), want)


def test_append_values_that_are_not_finite_and_zeros(hip_lib):
    ctx, new = [0, 8, 20, 0], [20, 4, 3, 5]
    s = Setup(ctx, new, 2, 32, 16)
    x = s.rng.standard_normal((s.tokens, 2, 32)).astype(np.float32)
    x[17, 0, 3] = np.nan          # request 0, its second block, head 0
    x[21, 1, 0] = -np.inf         # request 1, a block that holds tokens
    x[27:32] = 0.0                # request 3: a block of zeros
    cache, batch = s.cache(), s.batch()
    cache.append(batch, dev(x), dev(x))
    with np.errstate(all="ignore"):
        law.append(s.kc, s.ks, x, ctx, new, s.table, False)
    np.testing.assert_array_equal(cache.k_scales.cpu().numpy(), s.ks)
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)
    assert np.isnan(s.ks[s.table[0, 1], 0]) and np.isnan(s.ks[s.table[1, 0], 1])
    assert (s.ks[s.table[3, 0]] == 0).all() and not s.kc[s.table[3, 0], :, :5].any()
    # attention: NaN exactly where a row sees such a block
    q = dev(s.rng.standard_normal((s.tokens, 2, 32)).astype(np.float32))
    out = cache.attend(batch, q)
    bad = torch.isnan(out).any(-1).cpu().numpy()
    want = np.zeros((s.tokens, 2), bool)
    want[16:20, 0] = True         # positions of request 0 in or past its second block
    want[20:24, 1] = True
    np.testing.assert_array_equal(bad, want)
    assert torch.isnan(out).all(-1).cpu().numpy()[want].all()


def test_tokens_without_a_block_are_not_written(hip_lib):
    ctx, new, bs = [0, 0], [40, 20], 16
    s = Setup(ctx, new, 2, 64, bs, holes=[(0, 1)], width=2)
    x = s.rng.standard_normal((s.tokens, 2, 64)).astype(np.float32)
    cache, batch = s.cache(), s.batch()
    cache.append(batch, dev(x), dev(x))
    law.append(s.kc, s.ks, x, ctx, new, s.table, False)
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)
    k, _ = cache.read(dev(s.table), dev(np.zeros(2, np.int32)),
                      dev(np.array([0, 40, 60], np.int32)), 60, dtype="f32")
    # a hole (positions 16..31) and what lies past the table (32..39); request
    # 1 has both its blocks
    assert not k[16:40].any() and k[:16].any() and k[56:60].any()


# ------------------------------------------------------------------ attend

ATTENDS = {
    "one token alone": (lens((0, 1)), 4, 2, 64, 16, 0),
    "short": (lens((37, 1)), 32, 8, 128, 16, 0),
    "ragged step": (lens((0, 1), (1, 1), (15, 1), (16, 1), (63, 1), (64, 1), (65, 1), (700, 1)),
                    8, 2, 128, 16, 0),
    "absent requests": (lens((50, 0), (0, 0), (100, 1), (0, 0), (33, 2)), 8, 4, 64, 32, 0),
    "few tokens": (lens((300, 3), (129, 4), (0, 2)), 8, 2, 256, 64, 0),
    "wide heads": (lens((900, 1), (31, 1)), 16, 4, 256, 128, 0),
    "one kv head": (lens((200, 2), (17, 1)), 16, 1, 128, 32, 0),
    "many queries to a head": (lens((130, 1), (64, 2)), 40, 2, 64, 16, 0),
    "very many queries to a head": (lens((70, 2),), 142, 1, 64, 64, 0),
    "five to a head": (lens((333, 1), (10, 3)), 10, 2, 128, 64, 0),
    "own heads": (lens((257, 1), (99, 1)), 6, 6, 64, 128, 0),
    "prompt": (lens((0, 130),), 4, 1, 64, 64, 0),
    "prompts": (lens((0, 33), (0, 1), (0, 77), (0, 128), (0, 16)), 8, 2, 128, 32, 0),
    "chunk": (lens((200, 70),), 8, 2, 256, 64, 0),
    "mixed": (lens((500, 1), (70, 65), (0, 40), (12, 1), (64, 17)), 8, 4, 128, 16, 0),
    "window": (lens((300, 1), (40, 100), (0, 64), (5, 1)), 8, 4, 64, 32, 48),
    "window of one": (lens((77, 3), (0, 20)), 4, 2, 128, 16, 1),
    "window past all": (lens((77, 3), (0, 20)), 4, 2, 128, 16, 1 << 30),
    "small dims": (lens((100, 5), (3, 30)), 4, 2, 16, 16, 0),
    "odd dims": (lens((100, 1), (3, 30)), 6, 3, 80, 32, 20),
    "dims 96": (lens((640, 1), (30, 40)), 8, 2, 96, 64, 0),
    "long": (lens((20_011, 1), (5_000, 2)), 4, 1, 128, 64, 0),
    "long chunk": (lens((3_001, 50),), 2, 1, 64, 128, 0),
}


def attend_case(s, heads, window, dtype, q=None, strided=False, check=True):
    q = s.rng.standard_normal((s.tokens, heads, s.hd)) * 1.5 if q is None else q
    t = dev(q.astype(np.float32), TYPES[dtype])
    q = t.float().cpu().numpy()
    kw = {}
    if strided:
        wide = torch.full((s.tokens, heads + 1, s.hd + 16), 7.0, dtype=TYPES[dtype], device="cuda")
        wide[:, :heads, :s.hd] = t
        t = wide[:, :heads, :s.hd]
        kw["out"] = torch.zeros(s.tokens, heads + 2, s.hd + 8, dtype=TYPES[dtype],
                                device="cuda")[:, 1:heads + 1, :s.hd]
    scale = 1 / np.sqrt(s.hd)
    cache, batch = s.cache(), s.batch(heads, window)
    out, lse = cache.attend(batch, t, scale, return_lse=True, **kw)
    again, lse2 = cache.attend(batch, t, scale, return_lse=True)
    n = sum(s.new)                # rows past it are not written
    out, lse, again, lse2 = out[:n], lse[:n], again[:n], lse2[:n]
    assert torch.equal(torch.nan_to_num(out, 9.0), torch.nan_to_num(again, 9.0))
    assert torch.equal(torch.nan_to_num(lse, 9.0), torch.nan_to_num(lse2, 9.0))
    if not check:
        return out, lse
    o, l, ob, lb = law.attend(q, s.kc, s.vc, s.ks, s.vs, s.ctx, s.new, s.table,
                              float(np.float32(scale)), window, dtype, half_p=dtype != "f32")
    got, got_l = out.double().cpu().numpy(), lse.double().cpu().numpy()
    o, l, ob, lb = o[:n], l[:n], ob[:n], lb[:n]
    empty = np.isinf(l)
    np.testing.assert_array_equal(np.isneginf(got_l), empty)
    assert not got[empty].any()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(o))
    off = (np.abs(got - o) - ob)[~np.isnan(o)]
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:5].tolist())
    off = np.abs(got_l[~empty] - l[~empty]) - lb[~empty]
    assert (off <= 0).all(), float(off.max())
    return out, lse


@pytest.mark.parametrize("name", list(ATTENDS))
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attend_matches_64_bits(hip_lib, name, dtype):
    (ctx, new), heads, kv, hd, bs, window = ATTENDS[name]
    s = Setup(ctx, new, kv, hd, bs, seed=len(name), extra_rows=2)
    attend_case(s, heads, window, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hd,bs", [(128, 64), (64, 16), (256, 32), (48, 32)])
def test_attend_strided_queries_and_output(hip_lib, dtype, hd, bs):
    s = Setup([300, 0, 64], [1, 40, 2], 2, hd, bs)
    attend_case(s, 6, 0, dtype, strided=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 256, 32])
def test_attend_missing_blocks_and_empty_rows(hip_lib, dtype, hd):
    # request 0 lost blocks inside, request 1 all, request 2 (a prompt) its
    # first, so its early tokens see nothing; request 3's table is too narrow
    bs = 16
    ctx, new = [200, 40, 0, 160], [1, 1, 40, 60]
    s = Setup(ctx, new, 2, hd, bs, width=13,
              holes=[(0, 2), (0, 3), (0, 12), (1, 0), (1, 1), (1, 2), (2, 0)])
    out, lse = attend_case(s, 8, 0, dtype)
    assert torch.isneginf(lse[1]).all() and torch.isneginf(lse[2:18]).all()
    assert not out[1].any()


def test_attend_window_hides_a_block_that_is_not_finite(hip_lib):
    for hd in (64, 128, 256, 32):
        s = Setup([200, 100], [1, 40], 2, hd, 16)
        s.ks[s.table[0, 0]] = np.nan
        s.vs[s.table[0, 1]] = np.inf
        s.vs[s.table[1, 2]] = np.nan
        out, lse = attend_case(s, 4, 60, "bf16")
        # request 1's block 2 ends at position 47: tokens up to 106 see it
        bad = torch.isnan(out).any(-1).any(-1).cpu().numpy()
        np.testing.assert_array_equal(bad, [False] + [i <= 6 for i in range(40)])
        assert torch.isfinite(lse).all()


def test_attend_future_blocks_that_are_not_finite(hip_lib):
    # a chunk whose last block is NaN: only the rows that reach it are
    for hd in (64, 128, 256, 32):
        s = Setup([20], [60], 2, hd, 16)
        s.vs[s.table[0, 4], 1] = np.nan              # positions 64..79, head 1
        out, _ = attend_case(s, 8, 0, "f16", check=False)
        bad = torch.isnan(out).any(-1).cpu().numpy()
        want = np.zeros((60, 8), bool)
        want[44:, 4:] = True
        np.testing.assert_array_equal(bad, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
def test_attend_extreme_scores_and_scales(hip_lib, dtype, hd):
    # scores in the hundreds, value scales over twelve binary orders, blocks
    # of zeros, queries of zeros and tiny ones
    s = Setup([700, 0], [1, 50], 2, hd, 64)
    s.vs *= np.exp2(s.rng.integers(-6, 7, s.vs.shape)).astype(np.float32)
    s.vs[s.table[0, 3]] = 0.0
    s.ks[s.table[0, 5]] = 0.0
    q = s.rng.standard_normal((s.tokens, 8, hd)) * 20
    q[0, 1] = 0.0
    q[3] *= 1e-6
    q[4, 0] *= 60
    attend_case(s, 8, 0, dtype, q=q)


@pytest.mark.parametrize("heads,kv,ctx,new", [(16, 4, [0] * 60, [30] * 60),
                                              (16, 16, [i % 25 for i in range(200)], [2] * 200)])
def test_attend_f32_weights_keep_their_second_term(hip_lib, heads, kv, ctx, new):
    """Scores near 0 and few keys: what is left of the bound is the weights'
    own 21 bits, so that one weight that lost a unit of its first 11 shows.
    One in 2^13 is where that could happen."""
    s = Setup(ctx, new, kv, 64, 16, seed=5)
    attend_case(s, heads, 0, "f32", q=s.rng.standard_normal((s.tokens, heads, 64)) * 2.0 ** -9)


def test_attend_on_another_stream_and_in_a_graph(hip_lib):
    s = Setup([300, 10, 2000], [1, 30, 1], 2, 128, 32)
    cache, batch = s.cache(), s.batch(8)
    q = dev(s.rng.standard_normal((s.tokens, 8, 128)).astype(np.float32), torch.bfloat16)
    k = dev(s.rng.standard_normal((s.tokens, 2, 128)).astype(np.float32), torch.bfloat16)
    starts, cu = dev(np.array(s.ctx, np.int32)), dev(np.array([0, 1, 31, 32], np.int32))

    def step():
        batch.plan()
        cache.append(batch, k, k)
        out = cache.attend(batch, q)
        return out, cache.read(batch.block_table, starts, cu, 32)[0]

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    for i in range(4):
        held[0].zero_()
        held[1].zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_device_arrays_without_torch(hip_lib):
    s = Setup([70, 0], [1, 20], 2, 64, 16)
    put = DeviceArray.from_host
    cache = KvCache(put(s.kc), put(s.vc), put(s.ks), put(s.vs))
    batch = KvBatch(put(np.array(s.ctx, np.int32)), put(np.array(s.new, np.int32)), put(s.table),
                    16, tokens=s.tokens, max_new=20, heads=4, kv_heads=2).plan()
    q = s.rng.standard_normal((s.tokens, 4, 64)).astype(np.float32)
    x = s.rng.standard_normal((s.tokens, 2, 64)).astype(np.float16)
    cache.append(batch, put(x), put(x))
    out, lse = cache.attend(batch, put(q), return_lse=True)
    law.append(s.kc, s.ks, x.astype(np.float32), s.ctx, s.new, s.table, False)
    law.append(s.vc, s.vs, x.astype(np.float32), s.ctx, s.new, s.table, True)
    o, l, ob, lb = law.attend(q, s.kc, s.vc, s.ks, s.vs, s.ctx, s.new, s.table, 0.125, 0, "f32",
                              half_p=False)
    assert (np.abs(out.to_host() - o) <= ob).all() and (np.abs(lse.to_host() - l) <= lb).all()


def test_a_cache_past_four_gib(hip_lib):
    # 34,000 blocks of 128 x 8 x 128 bytes: 4.5 GB of key codes; the request's
    # blocks lie at both ends
    kv, hd, bs, pool = 8, 128, 128, 34_000
    g = torch.Generator(device="cuda").manual_seed(3)
    kc = torch.zeros((pool, kv, bs, hd), dtype=torch.int8, device="cuda")
    vc = torch.zeros((pool, kv, hd, bs), dtype=torch.int8, device="cuda")
    ks = torch.full((pool, kv), float("nan"), device="cuda")
    vs = torch.full((pool, kv), float("nan"), device="cuda")
    blocks = [0, pool - 1, 17_001, pool - 2, 1]
    table = dev(np.array([blocks], np.int32))
    n = bs * len(blocks) - 5
    x = torch.randn(2, n, kv, hd, generator=g, device="cuda")
    cache = KvCache(kc, vc, ks, vs)
    batch = KvBatch(dev(np.array([0], np.int32)), dev(np.array([n], np.int32)), table, bs,
                    tokens=n, max_new=n, heads=kv, kv_heads=kv).plan()
    cache.append(batch, x[0], x[1])
    k, v = cache.read(table, dev(np.array([0], np.int32)), dev(np.array([0, n], np.int32)), n,
                      dtype="f32")
    # a code is within half a step of its value, a step is its block's scale
    # (and both roundings of the law, 2^-22 of the value)
    for got, want, sc in ((k, x[0], ks), (v, x[1], vs)):
        step = sc[torch.tensor(blocks, device="cuda")].repeat_interleave(bs, 0)[:n, :, None]
        assert ((got - want).abs() <= step * 0.5 + want.abs() * 2.0 ** -22).all()
    q = torch.randn(n, kv, hd, generator=g, device="cuda")
    out = cache.attend(batch, q)
    s = torch.einsum("qhd,khd->hqk", q.double(), k.double()) / hd ** 0.5
    s.masked_fill_(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), -float("inf"))
    want = torch.einsum("hqk,khd->qhd", s.softmax(-1), v.double())
    # fp32 sums of at most 640 terms and 128-term scores below 2^4
    assert (out - want).abs().max() < 640 * 2 ** -24 * 8 + 128 * 2 ** -24 * 16 * 2 * 4


def test_results_on_a_stream_that_is_named(hip_lib):
    """Memory that a call makes belongs to the stream it was given."""
    s = Setup([300, 10, 900], [1, 30, 1], 2, 128, 32)
    cache, batch = s.cache(), s.batch(8)
    q = dev(s.rng.standard_normal((s.tokens, 8, 128)).astype(np.float32), torch.bfloat16)
    starts, cu = dev(np.array(s.ctx, np.int32)), dev(np.array([0, 1, 31, 32], np.int32))
    want = (*cache.attend(batch, q, return_lse=True), *cache.read(batch.block_table, starts, cu, 32))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for on in (side, side.cuda_stream, torch.cuda.current_stream(), 0):
        for _ in range(3):
            got = (*cache.attend(batch, q, return_lse=True, stream=on),
                   *cache.read(batch.block_table, starts, cu, 32, stream=on))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("hd", [64, 128, 256, 48])
def test_a_table_without_columns(hip_lib, hd):
    """No token has a block: nothing is written, and every row sees nothing."""
    s = Setup([0, 5, 0], [1, 0, 40], 2, hd, 16)
    cache = s.cache()
    b = KvBatch(dev(np.array(s.ctx, np.int32)), dev(np.array(s.new, np.int32)),
                torch.empty((3, 0), dtype=torch.int32, device="cuda"), 16, tokens=41, max_new=40,
                heads=4, kv_heads=2).plan()
    assert (b.slot_map == -1).all()
    x = dev(s.rng.standard_normal((41, 2, hd)).astype(np.float32))
    cache.append(b, x, x)
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)
    q = dev(s.rng.standard_normal((41, 4, hd)).astype(np.float32))
    out, lse = cache.attend(b, q, return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


def test_attend_more_items_than_a_grid_dimension(hip_lib):
    """128 query heads to a kv head: an item to a token, 66000 of them."""
    n, heads, hd, bs, window = 66_000, 128, 64, 128, 9
    g = torch.Generator(device="cuda").manual_seed(1)
    blocks = -(-n // bs)
    cache = KvCache(torch.randint(-127, 128, (blocks, 1, bs, hd), generator=g, device="cuda",
                                  dtype=torch.int8),
                    torch.randint(-127, 128, (blocks, 1, hd, bs), generator=g, device="cuda",
                                  dtype=torch.int8),
                    torch.full((blocks, 1), 0.01, device="cuda"),
                    torch.full((blocks, 1), 0.01, device="cuda"))
    batch = KvBatch(dev(np.array([0], np.int32)), dev(np.array([n], np.int32)),
                    torch.arange(blocks, dtype=torch.int32, device="cuda")[None], bs, tokens=n,
                    max_new=n, heads=heads, kv_heads=1, window=window).plan()
    q = torch.randn(n, heads, hd, generator=g, device="cuda", dtype=torch.bfloat16)
    out = cache.attend(batch, q)
    for row in (0, 8, 32_767, 65_535, 65_536, 65_999):
        at = torch.arange(max(0, row + 1 - window), row + 1, device="cuda")
        k = cache.k_codes[at // bs, 0, at % bs].double() * cache.k_scales[0, 0].double()
        v = cache.v_codes[at // bs, 0, :, at % bs].double() * cache.v_scales[0, 0].double()
        p = torch.softmax(q[row].double() @ k.t() / hd ** 0.5, -1)
        # bf16's rounding of the output, fp16's of the weights, fp32 scores
        bound = 2.0 ** -8 * (p @ v).abs() + 2.0 ** -10 * (p @ v.abs())
        assert ((out[row].double() - p @ v).abs() <= bound).all(), row


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 128), (256, 32)])
@pytest.mark.parametrize("window", [0, 100])
def test_attend_steps_where_the_window_or_the_table_bounds_the_work(hip_lib, dtype, hd, bs, window):
    """Steps of single tokens: long contexts behind a short window, and short
    ones on either side of a tile, with a block to a request."""
    ctx = [2900, 3, 64, 127, 1000] if window else [0, 3, 63, 64, 127, 128, 450]
    s = Setup(ctx, [1] * len(ctx), 2, hd, bs, seed=hd, holes=[(3, 0)])
    attend_case(s, 8, window, dtype)
