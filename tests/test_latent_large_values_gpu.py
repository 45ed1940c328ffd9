"""Means of values near the largest of their type, in both forms of latent
attention: the sums on the way to a mean stay in range where the mean does."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_amd import LatentCache  # noqa: E402
from tests.test_latent_gpu import Setup, dev  # noqa: E402
from tests.test_latent_rows_gpu import Rows  # noqa: E402

pytestmark = pytest.mark.gpu


def large(rng, shape):
    """Values in [2^126, 2^127.5), all of a channel of one sign, so that means are
    as large."""
    sign = np.where(rng.random(shape[-1]) < 0.5, -1.0, 1.0)
    return dev(sign * 2.0 ** (126 + 1.5 * rng.random(shape)), torch.bfloat16)


@pytest.mark.parametrize("rank,rope,heads", [(512, 64, 16), (512, 64, 40), (512, 64, 128),
                                             (256, 32, 16), (256, 32, 40), (256, 32, 128),
                                             (64, 16, 4)])
@pytest.mark.parametrize("ctx,new", [([300, 0], [1, 1]), ([4000], [1]), ([200], [40])])
def test_means_of_large_latents(hip_lib, rank, rope, heads, ctx, new):
    # The scores come from the key parts alone, and rise along the context, so that a
    # running maximum lags behind them.
    s = Setup(ctx, new, rank, rope, 16, heads)
    there = ~torch.isnan(s.rows[..., :1])
    s.rows[..., :rank] = torch.where(there, large(s.rng, tuple(s.rows.shape[:2]) + (rank,)), s.rows[..., :rank])
    s.q[..., :rank] = 0
    out, lse = LatentCache(s.rows, rank).attend(s.batch(), s.q, s.scale, return_lse=True)
    s.check(out, lse, heads_of=[0, heads - 1])


@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64), (128, 128), (24, 40)])
@pytest.mark.parametrize("ctx,new", [([300, 0], [1, 1]), ([4000], [3]), ([100], [200])])
@pytest.mark.parametrize("scale", [0.05, 0.3, -0.3])
def test_means_of_large_values(hip_lib, dk, dv, ctx, new, scale):
    s = Rows(ctx, new, dk, dv, 2)
    s.v = large(np.random.default_rng(1), tuple(s.v.shape))
    s.scale = scale
    s.check(*s.run(softmax_scale=scale))


@pytest.mark.parametrize("dk,dv", [(192, 128), (24, 40)])
def test_a_maximum_that_lags_behind(hip_lib, dk, dv):
    # Scores rise by a fifth of an octave a row: the reference is up to eight octaves
    # behind them when it moves.
    s = Rows([1500], [20], dk, dv, 2)
    s.k.zero_()
    s.q.zero_()
    s.q[..., 0] = 1
    s.k[..., 0] = dev(np.floor(np.arange(s.k.shape[0]) / 8)[:, None] * np.ones(2), torch.bfloat16)
    s.v = large(np.random.default_rng(2), tuple(s.v.shape))
    s.scale = 1.6 * np.log(2.0)
    s.check(*s.run(softmax_scale=s.scale))


def sized(rng, shape):
    """Values of both signs in [1/8, 15/8], bf16."""
    return dev(rng.choice([-1.0, 1.0], shape) * rng.integers(16, 240, shape) / 128, torch.bfloat16)


def same_multiple(got, power, rows):
    """The second results are 2^power times the first.  Sums stand at 2^-bits of
    themselves, bits = ceil(log2 rows) + 9 (rows that the call could see).  Where terms
    of theirs are below 2^-126, each of 2 rows products and additions is off by half of
    fp32's least step, 2^-150: by rows 2^(bits - 149) in an output, whose sum of weights
    is 1 or more, before it is rounded.  Two numbers so far from one another round to
    such as are a step of bf16 further apart at most (2^-7 of them)."""
    (out, lse), (out2, lse2) = got
    assert torch.equal(lse, lse2)
    want, off = out.double() * 2.0 ** power, (out2.double() - out.double() * 2.0 ** power).abs()
    if power < -60:
        bits = int(np.ceil(np.log2(rows))) + 9
        assert (off <= 2.0 ** -7 * want.abs() + 2 * rows * 2.0 ** (bits - 149)).all()
    else:
        assert (off == 0).all()


@pytest.mark.parametrize("power", [-100, -60, 60, 126])
@pytest.mark.parametrize("ctx,new", [([300, 0], [1, 1]), ([4000], [3]), ([70], [200])])
@pytest.mark.parametrize("rank,rope,heads", [(512, 64, 16), (512, 64, 128), (256, 32, 40), (64, 16, 4)])
def test_latents_times_a_power_of_two(hip_lib, rank, rope, heads, ctx, new, power):
    # (the scores are the key parts')
    s = Setup(ctx, new, rank, rope, 16, heads)
    s.rows.nan_to_num_(0.0)
    s.q[..., :rank] = 0
    s.rows[..., :rank] = sized(s.rng, tuple(s.rows.shape[:2]) + (rank,))
    batch, got = s.batch(), []
    for p in (0, power):
        s.rows[..., :rank] *= 2.0 ** p
        got.append(LatentCache(s.rows, rank).attend(batch, s.q, s.scale, return_lse=True))
    same_multiple(got, power, s.table.shape[1] * 16)


@pytest.mark.parametrize("power", [-100, -60, 60, 126])
@pytest.mark.parametrize("ctx,new", [([300, 0], [1, 1]), ([4000], [3]), ([100], [200])])
@pytest.mark.parametrize("dk,dv", [(192, 128), (96, 64), (128, 128), (24, 40)])
def test_values_times_a_power_of_two(hip_lib, dk, dv, ctx, new, power):
    s, got = Rows(ctx, new, dk, dv, 2), []
    s.v = sized(np.random.default_rng(1), tuple(s.v.shape))
    for p in (0, power):
        s.v = s.v * 2.0 ** p
        got.append(s.run())
    same_multiple(got, power, s.k.shape[0])
