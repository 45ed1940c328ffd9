"""Latent attention on the GPU with values at the ends of their types: rows that
are not finite under a negative scale, means of large values."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_latent_rows_gpu import Rows  # noqa: E402

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64), (24, 40)])
@pytest.mark.parametrize("bad", [INF, -INF])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("ctx,new,row", [(40, 1, 7), (40, 64, 7), (4000, 2, 1900)])
def test_a_negative_scale_hides_no_bad_key(hip_lib, dk, dv, bad, sign, ctx, new, row):
    # A score of either sign without end, of every token that there is: of weight 0
    # under one sign of the scale, and no finite number all the same.
    s = Rows([ctx], [new], dk, dv, 2)
    s.scale = -0.2
    s.k[row, 1, 3] = bad
    s.q[:, 1, 3] = sign
    out, lse = s.run(softmax_scale=-0.2)
    assert torch.isnan(out[:, 1]).all() and torch.isnan(lse[:, 1]).all()
    s.check(out, lse, heads_of=[0])
