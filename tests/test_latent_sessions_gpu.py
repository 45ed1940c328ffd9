"""The latent operators run together, as a serving program does."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import latent as law  # noqa: E402

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "latent_sessions.py"
    spec = importlib.util.spec_from_file_location("latent_sessions", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def host(t):
    return t.double().cpu().numpy()


def within(got, want, bound):
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all()


def test_sessions_mount_read_decode_and_harvest(hip_lib):
    m = example()
    sessions, prompt, steps = 5, 37, 6
    got = m.run(sessions=sessions, prompt=prompt, steps=steps)
    lengths, rotary = got["lengths"], got["rotary"]
    assert got["ctx"].tolist() == [n + prompt + steps for n in lengths]
    starts = torch.zeros(sessions, dtype=torch.int32, device="cuda")
    cu = torch.cat([starts[:1], got["ctx"].cumsum(0)]).int()
    for layer, cache in enumerate(got["caches"]):
        rows = host(cache.read(got["table"], starts, cu, int(cu[-1]), dtype="f32"))
        for s, n in enumerate(lengths):
            at, graft = int(cu[s]), host(got["grafts"][s][layer])
            np.testing.assert_array_equal(rows[at:at + n, :m.RANK], graft[:, :m.RANK])
            want, mass = law.turned(graft[:, None, m.RANK:], range(n), rotary.frequencies,
                                    rotary.magnitude, "half")
            within(rows[at:at + n, None, m.RANK:], want, law.turned_bound(want, mass, "bf16"))
        # the turn, turned back: both of a pair were rounded to bf16 (2^-8 of each at
        # most, 2^-8 of their hypotenuse together, which a turn keeps), beside two
        # turns in fp32, whose 18 units of 2^-24 are less than a sixteenth of it
        wrote, turn = host(got["wrote"][layer]), host(got["turn"][layer])
        np.testing.assert_array_equal(turn[..., :m.RANK], wrote[..., :m.RANK])
        a, b = np.split(wrote[..., m.RANK:], 2, -1)
        bound = np.hypot(a, b) * 2.0 ** -8 * (1 + 1 / 16)
        within(turn[..., m.RANK:], wrote[..., m.RANK:], np.concatenate([bound, bound], -1))
    # the prompt's attention of the last layer, over the keys and values it had
    r = got["read"]
    want, _, bound, _ = law.attend_rows(host(r["q"]), host(r["k"]), host(r["v"]), r["ctx"],
                                        [prompt] * sessions, r["cu"].tolist(), [0] * sessions,
                                        m.SCALE, 0, "bf16")
    within(host(r["out"]), want, bound)
    # and the last step's, over the cache
    table = got["table"].cpu().numpy()
    ctx = [n - 1 for n in got["ctx"].tolist()]
    rows = np.nan_to_num(host(got["caches"][-1].rows))
    want, _, bound, _ = law.attend(host(got["q"]), rows, m.RANK, ctx, [1] * sessions, table,
                                   m.SCALE, 0, "bf16")
    within(host(got["out"]), want, bound)
