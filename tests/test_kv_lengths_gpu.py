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
