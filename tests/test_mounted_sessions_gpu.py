"""The example that mounts grafts into the 8-bit cache and decodes on them."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "mounted_sessions.py"
    spec = importlib.util.spec_from_file_location("mounted_sessions", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_sessions_mount_decode_and_read_back(hip_lib):
    m = example()
    sessions, steps = 5, 6
    got = m.run(sessions=sessions, steps=steps)
    assert got["ctx"].tolist() == [n + steps for n in got["lengths"]]
    starts = torch.zeros(sessions, dtype=torch.int32, device="cuda")
    cu = torch.cat([starts[:1], got["ctx"].cumsum(0)]).int()
    for layer, cache in enumerate(got["caches"]):
        k, v = (t.double().cpu() for t in cache.read(got["table"], starts, cu, int(cu[-1]),
                                                     dtype="f32"))
        turn_k, turn_v = (t.double().cpu() for t in got["turn"][layer])
        for s, n in enumerate(got["lengths"]):
            at, end = int(cu[s]), int(cu[s + 1])
            for mine, turn, graft in ((k, turn_k, got["grafts"][s][0]),
                                      (v, turn_v, got["grafts"][s][1])):
                # a code is within half a step of its value; a held code that
                # follows a grown scale (the last block's) moves by another half
                # each time, steps times at most
                want = graft[layer].transpose(0, 1).double().cpu()
                step = mine[at:end].abs().amax() / 127
                off = (mine[at:at + n] - want).abs().amax()
                assert off <= step * (steps + 1) / 2 + 1e-3
                back = turn[s * steps:(s + 1) * steps]          # the same values in fp16
                assert torch.equal(back.half(), mine[at + n:end].half())
    # the last step's attention of the last layer, from the values read back
    group = m.HEADS // m.KV_HEADS
    q, out = got["q"].double().cpu(), got["out"].double().cpu()
    for s in range(sessions):
        at, end = int(cu[s]), int(cu[s + 1])
        for h in range(m.HEADS):
            kk, vv = k[at:end, h // group], v[at:end, h // group]
            p = torch.softmax(kk @ q[s, h] / np.sqrt(m.DIM), 0)
            bound = 2.0 ** -8 * (p @ vv).abs() + 2.0 ** -10 * (p @ vv.abs())
            assert ((out[s, h] - p @ vv).abs() <= bound).all()
