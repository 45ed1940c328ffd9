"""Prompts whose units are cut into parts, at every head_dim that the matrix
cores take: two parts, three (an odd one is left over where a block takes two
items), more, and several units beside each other."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import kv as law  # noqa: E402
from tests.test_kv_cache_gpu import ATTENDS, TYPES, Setup, dev  # noqa: E402

pytestmark = pytest.mark.gpu


def check(s, heads, dtype, window=0, spread=1.5):
    """Against 64 bits, within the bound of weights of fp32 (2^-20); twice."""
    t = dev((s.rng.standard_normal((s.tokens, heads, s.hd)) * spread).astype(np.float32),
            TYPES[dtype])
    scale = 1 / np.sqrt(s.hd)
    cache, batch = s.cache(), s.batch(heads, window)
    out, lse = cache.attend(batch, t, scale, return_lse=True)
    again = cache.attend(batch, t, scale)
    n = sum(s.new)
    assert torch.equal(out[:n], again[:n])
    o, l, ob, lb = law.attend(t.float().cpu().numpy(), s.kc, s.vc, s.ks, s.vs, s.ctx, s.new, s.table,
                              float(np.float32(scale)), window, dtype, half_p=False)
    off = np.abs(out[:n].double().cpu().numpy() - o[:n]) - ob[:n]
    assert (off <= 0).all(), (float(off.max()), np.argwhere(off > 0)[:4].tolist())
    seen = ~np.isinf(l[:n])
    got = lse[:n].double().cpu().numpy()
    np.testing.assert_array_equal(np.isneginf(got), ~seen)
    assert (np.abs(got[seen] - l[:n][seen]) <= lb[:n][seen]).all()
    return batch


PARTS = {
    # ctx, new, block tokens, window; the units of 32 tokens that are cut
    "two parts": ([700], [40], 64, 0, 2),
    "three parts": ([1200], [60], 32, 0, 2),
    "more parts": ([1900], [33], 128, 0, 2),
    "units of unlike parts": ([1500, 30, 650, 0], [140, 1, 50, 70], 64, 0, 7),
    "a window": ([1500, 900], [90, 20], 16, 900, 4),
}


@pytest.mark.parametrize("name", list(PARTS))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_units_that_are_cut(hip_lib, dtype, hd, name):
    ctx, new, bs, window, cut = PARTS[name]
    s = Setup(ctx, new, 2, hd, bs, seed=hd + len(name))
    # value scales of several orders: the parts' sums are in unlike units
    s.vs *= np.exp2(s.rng.integers(-9, 10, s.vs.shape)).astype(np.float32)
    batch = check(s, 8, dtype, window)
    joins = int(batch._work[16:20].view(torch.int32))
    assert joins == cut


@pytest.mark.parametrize("name", list(ATTENDS))
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_outputs_within_the_bound_of_fp32_weights(hip_lib, name, dtype):
    (ctx, new), heads, kv, hd, bs, window = ATTENDS[name]
    check(Setup(ctx, new, kv, hd, bs, seed=len(name) + 1, extra_rows=1), heads, dtype, window)
