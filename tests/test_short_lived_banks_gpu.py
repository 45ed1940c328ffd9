"""Banks that live for one route, one after another: memory that the last one
freed holds its route's list entries, which the next one's first route must not
take for its own."""

import numpy as np
import pytest

import oracle
from graftrepository_amd import MlaNodeBank

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,dim,nq,k", [(3000, 64, 8, 6), (700, 96, 40, 4), (5000, 32, 1, 16)])
def test_a_bank_after_another(hip_lib, n, dim, nq, k):
    rng = np.random.default_rng(n)
    rows = rng.standard_normal((n, dim)).astype(np.float32)
    qs = rng.standard_normal((nq, dim)).astype(np.float32)
    sides = [(r, q, oracle.mla_route(r, q, k)[:2]) for r, q in ((rows, qs), (np.abs(rows), -np.abs(qs)))]
    for i in range(40):
        r, q, (ids, scores) = sides[i % 2]
        with MlaNodeBank(r) as bank:
            got = bank.route(q, k)
        np.testing.assert_array_equal(got.ids, ids)
        np.testing.assert_array_equal(got.scores.view(np.uint32), scores.view(np.uint32))
