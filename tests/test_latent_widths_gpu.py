"""Caches of both matrix-core widths on one batch, whose schedule has a plan for each."""

import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import LatentCache  # noqa: E402
from tests.test_latent_gpu import Setup  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [16, 40])
def test_each_width_follows_its_own_plan(hip_lib, heads):
    # 1250 tiles of 32 rows: a run has four at least, and one block to a CU (rank 512)
    # makes 256 runs of them, two (rank 256) 313
    big, small = (Setup([40_000, 3], [1, 1], rank, rope, 64, heads)
                  for rank, rope in ((512, 64), (256, 32)))
    assert (big.table == small.table).all()
    batch = big.batch()
    caches = [LatentCache(s.rows, s.rank) for s in (big, small)]
    for _ in range(2):
        for s, cache in zip((big, small), caches):
            out, lse = cache.attend(batch, s.q, s.scale, return_lse=True)
            s.check(out, lse, heads_of=[0, heads - 1])
            alone, lse2 = cache.attend(s.batch(), s.q, s.scale, return_lse=True)
            assert torch.equal(out, alone) and torch.equal(lse, lse2)
