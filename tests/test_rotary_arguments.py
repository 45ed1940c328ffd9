"""Arguments of a rotation that have no frequencies or no inverse."""

import ctypes

import pytest

import graftrepository_amd as g
from tests.test_rotary import rotary_desc

INF = float("inf")


@pytest.mark.parametrize("kw", [
    dict(scaling="factors", factors=[1.0] * 7 + [0.0]), dict(scaling="base", factor=1e-300),
    dict(scaling="base", factor=1e300), dict(scaling="yarn", factor=2.0, trained=INF),
    dict(scaling="smooth", factor=2.0, trained=INF), dict(scaling="smooth", fast=INF),
    dict(scaling="yarn", fast=INF), dict(scaling="yarn", slow=float("nan")),
])
def test_no_frequencies(kw):
    with pytest.raises(ValueError):
        g.Rotary(16, **kw)


def test_a_magnitude_without_an_inverse():
    lib = g.load()

    def rotate(**kw):
        return lib.grm_hip_rotate(ctypes.byref(rotary_desc(**kw)), None, 0, 64, 64, None, 64, 64,
                                  None, 0, 1, 64, 0, None)
    assert rotate(magnitude=1e-39) == 0
    assert rotate(magnitude=1e-39, inverse=1) == -1
    assert b"magnitude" in lib.grm_hip_last_error()
    assert rotate(magnitude=1e30, inverse=1) == 0
