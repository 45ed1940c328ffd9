"""Lengths on the device that say more than a batch has rows or its table has
places for: what has a row is served, and nothing else is touched."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch  # noqa: E402
from oracle import kv as law  # noqa: E402
from tests.test_kv_cache_gpu import Setup, dev  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,tokens", [([10, 8, 1], 10), ([10, 8, 1], 9), ([40, 3, 70], 41),
                                        ([5, 0, 6], 3), ([1, 1, 1], 1)])
def test_more_tokens_than_rows(hip_lib, new, tokens):
    """Blocks of tokens past the last row are in no list: what memory the
    schedule is in is not taken for one."""
    s = Setup([20, 7, 0], new, 2, 64, 16, seed=tokens)
    b = KvBatch(dev(np.array(s.ctx, np.int32)), dev(np.array(new, np.int32)), dev(s.table), 16,
                tokens=tokens, max_new=max(new), heads=4, kv_heads=2)
    b._work.fill_(0x11)
    b.plan()
    cache = s.cache()
    x = s.rng.standard_normal((tokens, 2, 64)).astype(np.float32)
    cache.append(b, dev(x), dev(x))
    have, left = [], tokens                  # the rows are dealt in request order
    for n in new:
        have.append(max(0, min(n, left)))
        left -= have[-1]
    law.append(s.kc, s.ks, x, s.ctx, have, s.table, False)
    law.append(s.vc, s.vs, x, s.ctx, have, s.table, True)
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)
    np.testing.assert_array_equal(cache.v_codes.cpu().numpy(), s.vc)
    np.testing.assert_array_equal(cache.k_scales.cpu().numpy(), s.ks)
    q = dev(s.rng.standard_normal((tokens, 4, 64)).astype(np.float32))
    out, lse = cache.attend(b, q, return_lse=True)
    # requests that are whole: the others' later tokens have no row
    whole = [n if n == h else 0 for n, h in zip(new, have)]
    o, l, ob, lb = law.attend(q.cpu().numpy(), s.kc, s.vc, s.ks, s.vs, s.ctx, whole, s.table, 0.125,
                              0, "f32", half_p=False)
    n = sum(whole)
    assert (np.abs(out[:n].cpu().numpy() - o[:n]) <= ob[:n]).all()


def test_lengths_whose_sum_passes_32_bits(hip_lib):
    """Rows past the batch's stay past its end, whatever their sum is."""
    far = (1 << 30) - 256
    new = [2, far, far, far, 1, 1]
    s = Setup([20, 0, 0, 0, 5, 9], [2, 0, 0, 0, 1, 1], 2, 64, 16)
    b = KvBatch(dev(np.array(s.ctx, np.int32)), dev(np.array(new, np.int32)), dev(s.table), 16,
                tokens=7, max_new=1, heads=4, kv_heads=2).plan()
    cu = b.cu_new.cpu().numpy()
    assert cu[1] == 2 and (cu[2:] > 7).all() and cu[2] == 2 + far
    cache = s.cache()
    x = s.rng.standard_normal((7, 2, 64)).astype(np.float32)
    cache.append(b, dev(x), dev(x))
    lens = [2, 5, 0, 0, 0, 0]                # five tokens of the long request have rows
    law.append(s.kc, s.ks, x, s.ctx, lens, s.table, False)
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)
    q = dev(s.rng.standard_normal((7, 4, 64)).astype(np.float32))
    out = torch.full_like(q, 7.0)
    cache.attend(b, q, out=out)
    assert not (out[:2] == 7.0).any() and (out[2:] == 7.0).all()


def scratch_of(s, heads, tokens=None, max_new=None, window=0, width=None):
    """(bytes of scratch, the batch) of a plan."""
    table = dev(s.table if width is None else s.table[:, :width])
    b = KvBatch(dev(np.array(s.ctx, np.int32)), dev(np.array(s.new, np.int32)), table, s.bs,
                tokens=s.tokens, max_new=max(s.new), heads=heads, kv_heads=s.kv,
                window=window).plan()
    cache = s.cache()
    cache.attend(b, torch.zeros(s.tokens, heads, s.hd, device="cuda"))
    return b._scratch[s.hd], b


@pytest.mark.parametrize("hd,kv,heads", [(128, 8, 32), (256, 4, 16), (64, 2, 64)])
def test_short_prompts_need_no_scratch_for_parts(hip_lib, hd, kv, heads):
    """A unit of at most eight tiles is never cut: a prompt whose table, or whose
    window, holds no more pays for no parts."""
    step, _ = scratch_of(Setup([100], [1], kv, hd, 64, width=8), heads)
    parts = 4 * 128 * (hd + 3) * kv                       # bytes of one, of every kv head
    assert scratch_of(Setup([100], [20], kv, hd, 64, width=8), heads)[0] <= step
    assert scratch_of(Setup([5000], [20], kv, hd, 64), heads, window=200)[0] <= step
    # and of longer ones for as many as the batch can make
    got, _ = scratch_of(Setup([1000], [20], kv, hd, 64), heads)
    units = -(-20 * (heads // kv) // 128) + 1
    assert step < got <= step + units * 3 * parts         # 17 tiles: three parts a unit


@pytest.mark.parametrize("window", [0, 700])
def test_tiles_past_the_table_are_not_looked_at(hip_lib, window):
    """Lengths far past the table's places: the tokens see what has a block, and
    the schedule ends there."""
    s = Setup([160, 100, 130], [1, 40, 20], 2, 64, 16)
    ctx = [160, 1 << 29, 130]
    b = KvBatch(dev(np.array(ctx, np.int32)), dev(np.array(s.new, np.int32)), dev(s.table), 16,
                tokens=s.tokens, max_new=40, heads=4, kv_heads=2, window=window).plan()
    units, tiles, items = b._work[4:16].view(torch.int32).tolist()
    assert units == 1 and tiles <= -(-s.width * 16 // 64) and items <= 4
    q = s.rng.standard_normal((s.tokens, 4, 64))
    t = dev(q.astype(np.float32))
    out, lse = s.cache().attend(b, t, 0.125, return_lse=True)
    # request 1 sees its table's blocks, or with a window none
    shown = [160, s.width * 16, 130]
    new = [1, 0, 20]
    rows = np.r_[0, 41:61]
    o, l, ob, lb = law.attend(t.cpu().numpy()[rows], s.kc, s.vc, s.ks, s.vs, shown, new, s.table,
                              0.125, window, "f32", half_p=False)
    assert (np.abs(out.cpu().numpy()[rows] - o) <= ob).all()
    if window:
        assert not out[1:41].any() and torch.isneginf(lse[1:41]).all()
    else:
        assert torch.isfinite(lse[1:41]).all() and out[1:41].any()
