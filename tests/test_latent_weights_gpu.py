"""Absorbed attention of 16 columns and less rounds its weights in two terms: outputs
are the means rounded once, whatever they cancel to."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import LatentCache  # noqa: E402
from oracle import latent as law  # noqa: E402
from tests.test_latent_gpu import Setup, host  # noqa: E402

pytestmark = pytest.mark.gpu
# The first bf16 term is cut (off by a step, 2^-7), the second rounds the rest (2^-8 of
# it); fp16 terms are rounded both (2^-11 each).
TWO = {"bf16": 2.0 ** -15, "f16": 2.0 ** -22}


@pytest.mark.parametrize("rank,rope", [(512, 64), (256, 32)])
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("ctx,new,heads", [([20, 3], [1, 1], 16), ([2000], [1], 16), ([40], [4], 4)])
def test_weights_in_two_terms(hip_lib, rank, rope, name, ctx, new, heads):
    s = Setup(ctx, new, rank, rope, 16, heads, name)
    s.q[..., :rank + rope - 4] = 0     # four terms to a score: the others add zeros
    out = host(LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale))
    rows, q, row = np.nan_to_num(host(s.rows)), host(s.q), 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        keys, _ = law.gather(rows, s.table[r], range(c + n))
        for i in range(n):
            for h in range(heads):
                k = keys[:c + i + 1]
                want, _, bound, _ = law.attend_one(q[row, h], k, k[:, :rank], s.scale, TWO[name],
                                                   name, 4)
                assert (np.abs(out[row, h] - want) <= bound).all()
            row += 1
