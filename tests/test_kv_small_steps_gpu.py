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


@pytest.mark.parametrize("heads", [2, 32, 64, 256, 260])
@pytest.mark.parametrize("hd", [128, 48])
def test_a_step_that_may_bring_no_token(hip_lib, heads, hd):
    """max_new = 0 with rows to spare: nothing to attend, whatever the group."""
    s = Setup([40, 3], [0, 0], 2, hd, 16, extra_rows=3)
    cache, batch = s.cache(), s.batch(heads)
    q = torch.randn(3, heads, hd, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 7.0)
    cache.append(batch, q[:, :2], q[:, :2])
    cache.attend(batch, q, out=out)
    assert (out == 7.0).all()
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), s.kc)


@pytest.mark.parametrize("tokens", [0, 5, 9000])
def test_a_batch_without_requests(hip_lib, tokens):
    """The plan writes its outputs all the same: sums, rows without a slot, and
    the free list's head, from which the next step goes on."""
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    b = KvBatch(none, none, none.view(0, 4), 16, tokens=tokens, max_new=1, heads=2, kv_heads=2,
                free_list=dev(np.arange(9, dtype=np.int32)),
                free_head=dev(np.array([3], np.int32)))
    for a in (b.cu_new, b.slot_map, b.positions, b.free_head_out):
        a.fill_(77)
    b.plan()
    assert b.cu_new.tolist() == [0] and b.free_head_out.tolist() == [3]
    assert (b.slot_map == -1).all() and (b.positions == -1).all()
    s = Setup([0], [1], 2, 64, 16)
    cache = s.cache()
    x = torch.randn(tokens, 2, 64, device="cuda")
    cache.append(b, x, x)
    assert cache.attend(b, x, out=torch.full_like(x, 7.0)).eq(7.0).all()
    b.advance()
    assert b.free_head.tolist() == [3]
