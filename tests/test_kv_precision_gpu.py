"""How many bits the 8-bit cache's attention keeps where a plain form in fp32
keeps them: weights whose products cancel, queries whose channels are of very
unlike size, value scales far from 1."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import kv as law  # noqa: E402
from tests.test_kv_cache_gpu import TYPES, Setup, dev  # noqa: E402

pytestmark = pytest.mark.gpu


def attend(s, q, heads, dtype, window=0):
    """(out, lse) in fp64 on the host, and the queries' values as held."""
    t = dev(q.astype(np.float32), TYPES[dtype])
    out, lse = s.cache().attend(s.batch(heads, window), t, 1 / np.sqrt(s.hd), return_lse=True)
    return out.double().cpu().numpy(), lse.double().cpu().numpy(), t.float().cpu().numpy()


def within(s, got, q, heads, dtype, window=0):
    """Against 64 bits, within the bound of fp32 weights (whole ones: 2^-20)."""
    o, l, ob, lb = law.attend(q, s.kc, s.vc, s.ks, s.vs, s.ctx, s.new, s.table,
                              float(np.float32(1 / np.sqrt(s.hd))), window, dtype, half_p=False)
    off = np.abs(got[0] - o) - ob
    assert (off <= 0).all(), (float((off / ob).max()), np.argwhere(off > 0)[:4].tolist())
    assert (np.abs(got[1] - l) <= lb).all()


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_outputs_keep_the_weights_second_term(hip_lib, dtype, hd, new):
    """Values that cancel but for the small difference of two blocks' scales:
    weights of 11 bits are off by 2^-12 of what cancels, several times the
    bound, in which the output's own rounding is small."""
    s = Setup([32], [new], 2, hd, 16, seed=hd + new)
    a, b = s.table[0, :2]
    s.vc[b] = -s.vc[a]
    s.vc[s.table[0, 2:4]] = 0                      # the new tokens' own values
    s.vs[a] = s.vs[b] * np.float32(1 + 2.0 ** -10)
    q = np.zeros((s.tokens, 8, hd))
    got = attend(s, q, 8, dtype)
    within(s, got, got[2], 8, dtype)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_queries_of_unlike_channels_keep_their_bits(hip_lib, dtype, hd, new):
    """One channel far above the others, and no key has anything in it: the
    scores are the others' alone, with all their bits."""
    s = Setup([100], [new], 2, hd, 16, seed=hd + new)
    s.kc[:, :, :, 5] = 0
    q = s.rng.standard_normal((s.tokens, 8, hd)) * 2
    q[..., 5] = 2.0 ** (15 if dtype == "f16" else 24)
    got = attend(s, q, 8, dtype)
    rest = got[2].copy()
    rest[..., 5] = 0.0
    within(s, got, rest, 8, dtype)


@pytest.mark.parametrize("new", [1, 64])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
def test_fp32_weights_are_whole(hip_lib, hd, new):
    """Rows that see one token: the output is its code times its scale, of 31
    bits.  A sum of exact products is rounded once or, if the matrix core cuts
    instead, off by a unit at most; the steps after it are by powers of two."""
    ctx = [16 * 30 - 1] * 40
    s = Setup(ctx, [new if r % 8 == 0 else 1 for r in range(40)], 2, hd, 16, seed=hd + new)
    s.vs *= np.exp2(s.rng.integers(-3, 4, s.vs.shape)).astype(np.float32)
    q = s.rng.standard_normal((s.tokens, 4, hd))
    got, _, _ = attend(s, q, 4, "f32", window=1)
    row = 0
    for r, n in enumerate(s.new):
        for i in range(n):
            p = s.ctx[r] + i
            b = s.table[r, p // 16]
            want = s.vc[b, :, :, p % 16].astype(np.float64) * s.vs[b][:, None].astype(np.float64)
            want = np.repeat(want, 2, 0)
            assert (np.abs(got[row] - want) <= np.abs(want) * 2.0 ** -23).all()
            row += 1


@pytest.mark.parametrize("power", [-100, -40, 40])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_value_scales_times_a_power_of_two(hip_lib, dtype, hd, new, power):
    """All value scales times 2^n give the outputs times 2^n, to the bit."""
    s = Setup([200], [new], 2, hd, 32, seed=hd + new)
    s.vs = np.where(np.isnan(s.vs), s.vs, np.float32(1.0) + np.abs(s.vs)).astype(np.float32)
    q = s.rng.standard_normal((s.tokens, 4, hd))
    plain = attend(s, q, 4, dtype)
    s.vs *= np.float32(2.0) ** power
    scaled = attend(s, q, 4, dtype)
    np.testing.assert_array_equal(scaled[0], plain[0] * 2.0 ** power)
    np.testing.assert_array_equal(scaled[1], plain[1])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_values_do_not_overflow_before_they_are_means(hip_lib, dtype, hd, new):
    """Sums of many values near fp32's largest pass it, their mean does not."""
    s = Setup([3000, 700], [new, 1], 2, hd, 64, seed=hd + new)
    s.vs *= np.float32(2.0) ** 119                 # values up to 2^127
    s.vs = np.minimum(s.vs, np.float32(2.0) ** 119)
    q = s.rng.standard_normal((s.tokens, 4, hd)) * 0.1
    got = attend(s, q, 4, dtype)
    assert np.isfinite(got[0]).all()
    within(s, got, got[2], 4, dtype)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_queries_that_are_not_finite(hip_lib, dtype, hd, new):
    """They make their own row and head NaN, and no other."""
    s = Setup([130, 20], [new, 1], 2, hd, 16, seed=hd)
    q = s.rng.standard_normal((s.tokens, 8, hd))
    q[0, 1, 3], q[new, 6, hd - 1], q[new // 2, 5, 0] = np.nan, np.inf, -np.inf
    out, lse, _ = attend(s, q, 8, dtype)
    bad = np.zeros((s.tokens, 8), bool)
    bad[0, 1] = bad[new, 6] = bad[new // 2, 5] = True
    np.testing.assert_array_equal(np.isnan(out).all(-1), bad)
    np.testing.assert_array_equal(np.isnan(out).any(-1), bad)
