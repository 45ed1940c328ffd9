"""Calls of more rows than one launch has room for: refused by the library, with its
message, before anything is read; rotations go on in further launches."""

import ctypes

import pytest

import graftrepository_amd as g
from tests.test_rotary import latent_desc, one_head

MOST = (2 ** 32 - 1) // 256          # blocks of 256 threads in a launch's first dimension


def refused(rc):
    assert rc == -1
    assert b"too many rows for one call" in g.load().grm_hip_last_error()


@pytest.mark.parametrize("rank,rows,heads", [(64, 128 * (MOST // 32) + 1, 64), (64, 1 << 29, 16),
                                             (48, MOST + 1, 1)])
def test_expansions(rank, rows, heads):
    refused(g.load().grm_hip_latent_expand(
        ctypes.byref(latent_desc(rank=rank)), 0x1000, heads, 64, 64, 0x1000, 4, 3, 0x1000, 0x1000,
        rows, 0x1000, 0x1000, None))


def test_reads_and_appends():
    lib = g.load()
    refused(lib.grm_hip_latent_read(ctypes.byref(latent_desc()), 0x1000, 4, 3, 0x1000, 0x1000,
                                    16 * MOST + 1, 0, 0x1000, None))
    batch = one_head(tokens=(256 * MOST) // 36 + 1)
    refused(lib.grm_hip_latent_append(ctypes.byref(latent_desc(rank=512, rope=64)),
                                      ctypes.byref(batch), None, 0x1000, 0x1000, 0, 512, 64, None))


def test_plain_attention():
    lib, batch = g.load(), one_head(tokens=MOST + 1)
    refused(lib.grm_hip_latent_attend(ctypes.byref(latent_desc()), ctypes.byref(batch), 0x1000,
                                      1 << 40, 0x1000, 384, 96, 0x2000, 256, 64, None, 1.0, None, 0,
                                      None))
    for dk, stride in ((64, 64), (192, 1 << 25)):
        refused(lib.grm_hip_rows_attend(ctypes.byref(batch), 0x1000, 1 << 40, 1, dk, 128, 0x1000, 256,
                                        64, 0x1000, stride, 64, 0x1000, 256, 64, 5, 0x1000, None,
                                        0x1000, 256, 64, None, 1.0, None, 0, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [6, 16])
@pytest.mark.parametrize("in_place", [False, True])
def test_more_rows_than_a_launch_are_turned(hip_lib, dim, in_place):
    torch = pytest.importorskip("torch")
    n = MOST + 700
    gen = torch.Generator(device="cuda")
    gen.manual_seed(dim)
    x = torch.randn(n, 1, dim, generator=gen, device="cuda").half()
    positions = torch.randint(0, 100_000, (n,), generator=gen, device="cuda", dtype=torch.int32)
    rotary = g.Rotary(dim)
    want = torch.cat([rotary.apply(a, p) for a, p in zip(x.split(1 << 22), positions.split(1 << 22))])
    out = rotary.apply(x, positions, out=x if in_place else None)
    assert torch.equal(out, want)
