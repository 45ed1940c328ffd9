"""Scratch of attention over dense rows: no more than its parts take, and none where
no unit can be cut."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch  # noqa: E402
from tests.test_latent_rows_gpu import Rows, ints  # noqa: E402

pytestmark = pytest.mark.gpu


def scratch(batch, dk, dv):
    got = ctypes.c_uint64()
    assert batch._lib.grm_hip_rows_attend_bytes(batch._ref, dk, dv, ctypes.byref(got)) == 0
    return got.value


@pytest.mark.parametrize("heads", [3, 40, 100, 128, 300])
def test_at_most_sixteen_parts_to_a_cu(hip_lib, heads):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for tokens in (600, 20_000):
        batch = KvBatch(ints([3000]), ints([tokens]), ints([[0]]), 64, tokens=tokens, max_new=tokens,
                        heads=heads, kv_heads=1, latent=True)
        assert 0 < scratch(batch, 96, 64) <= 16 * cus * 128 * (64 + 2) * 4
    s = Rows([3000], [600], 96, 64, heads)
    s.check(*s.run(), heads_of=[heads - 1])


def test_as_many_heads_as_blocks_cut_nothing(hip_lib):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for heads in (2 * cus, 2 * cus + 8):
        s = Rows([700, 0], [70, 200], 96, 64, heads)
        b = s.batch()
        assert scratch(b, 96, 64) == 0
        s.check(*s.run(), heads_of=[0, heads - 1])
