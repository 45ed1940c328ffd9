"""Tensors with forward-mode tangents, which have no requires_grad: refused, since a
result would be without its derivative."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as forward  # noqa: E402

from graftrepository_amd import (KvBatch, KvCache, LatentCache, Rotary,  # noqa: E402
                                 attend_rows)
from graftrepository_amd import kv_cache as kc  # noqa: E402
from tests.test_kv_cache import fake  # noqa: E402


def dual(x):
    return forward.make_dual(x, torch.ones_like(x))


def test_a_tangent_is_refused():
    x = torch.zeros(3, 2, 16)
    with forward.dual_level():
        d = dual(x)
        for a in (d, d[:, :1].expand(3, 2, 16), d * 2):
            with pytest.raises(ValueError, match="tangent"):
                kc._rows(a, "q", (3, 2, 16))
        with pytest.raises(ValueError, match="tangent"):
            Rotary(16).apply(d, fake((3,), np.int32))
        with pytest.raises(ValueError, match="tangent"):
            LatentCache(fake((4, 16, 96), np.float16), 64).expand(
                dual(torch.zeros(4, 64, 64)), 32, fake((3, 4), np.int32), fake((3,), np.int32),
                fake((4,), np.int32), 5)
        # without one it goes on to the other checks, as do arrays that are not torch's
        for a in (x, forward.unpack_dual(d).primal):
            with pytest.raises(ValueError, match="GPU"):
                kc._rows(a, "q", (3, 2, 16))
        assert kc._rows(fake((3, 2, 16), np.float16), "q", (3, 2, 16))[1] == "f16"
    with pytest.raises(ValueError, match="GPU"):
        kc._rows(x, "q", (3, 2, 16))


@pytest.mark.gpu
def test_calls_with_a_tangent_are_refused(hip_lib):
    def zeros(*shape, dtype=torch.float16):
        return torch.zeros(shape, device="cuda", dtype=dtype)

    def ints(*a):
        return torch.tensor(a, device="cuda", dtype=torch.int32)
    cache = LatentCache(zeros(2, 16, 288), 256)
    kv = KvCache(zeros(2, 1, 16, 64, dtype=torch.int8), zeros(2, 1, 64, 16, dtype=torch.int8),
                 zeros(2, 1, dtype=torch.float32), zeros(2, 1, dtype=torch.float32))
    batch = KvBatch(ints(0), ints(3), ints(0).view(1, 1), 16, tokens=3, max_new=3, heads=2,
                    kv_heads=1, latent=True).plan()
    latent, part, q = zeros(3, 256), zeros(3, 32), zeros(3, 2, 288)
    k, v, cu = zeros(3, 1, 64), zeros(3, 2, 64), ints(0, 3)
    q2, k2 = zeros(3, 2, 96), zeros(3, 2, 96)
    calls = [(cache.append, (batch, latent, part), (1, 2)), (cache.attend, (batch, q, 1.0), (1,)),
             (kv.append, (batch, k, k), (1, 2)), (kv.attend, (batch, zeros(3, 2, 64)), (1,)),
             (attend_rows, (batch, q2, k2, v, cu), (1, 2, 3)),
             (Rotary(32).apply, (part.unsqueeze(1), batch.positions), (0,))]
    for call, args, which in calls:
        for i in which:
            with forward.dual_level():
                with pytest.raises(ValueError, match="tangent"):
                    call(*args[:i], dual(args[i]), *args[i + 1:])
                call(*args)
