"""Steps of the 8-bit cache with nothing in them, or less than they allow, and
batches that end before the work that reads them."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import KvBatch  # noqa: E402
from tests.test_kv_cache_gpu import Setup, dev  # noqa: E402

pytestmark = pytest.mark.gpu


def test_a_batch_dropped_while_another_stream_reads_it(hip_lib):
    """Its memory is not handed out before that stream is through."""
    s = Setup([300, 10, 900], [1, 1, 1], 2, 64, 16)
    cache, side = s.cache(), torch.cuda.Stream()
    b = s.batch(4)
    q = torch.randn(3, 4, 64, device="cuda")
    want = cache.attend(b, q)
    torch.cuda.synchronize()
    size, at = b._work.nbytes, b._work.data_ptr()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    got = cache.attend(b, q, stream=side)
    del b
    others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    assert at not in [o.data_ptr() for o in others]
    torch.cuda.synchronize()
    assert torch.equal(got, want)
