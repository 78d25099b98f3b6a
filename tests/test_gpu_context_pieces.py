"""Linear attention whose sequences are cut into pieces, with the states in place (s1 = s0): the first piece starts from the
state that the call was given, whenever the last one stores its own."""
import numpy as np
import pytest

import context_ref as R
from test_gpu_context import LaCase, say

pytestmark = pytest.mark.gpu


def in_place(c):
    """c's call over its own s0; the workspace is of the pieces' size."""
    assert c.H.lib().bnh_linattn_work_bytes(c.args(), c.T, len(c.lens)) > 0, "one piece only"
    c.ds1 = c.ds0
    c.run()
    return c.do.get(), c.ds0.numpy()


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("lens,heads,dk,dv", [([600, 300, 257, 256, 1, 0], 4, 32, 48), ([1000], 3, 64, 130),
                                              ([129, 640], 2, 100, 24)], ids=str)
def test_in_place(hip, f16, lens, heads, dk, dv):
    """Against the definition: sequences of several pieces, of one that is full, of one row and of none."""
    say(f"la in place lens {lens} dk {dk} dv {dv} f16 {f16}")
    c = LaCase(hip, lens, heads, heads, heads, heads, dk, dv, f16, gscale=0.1, seed=dk)
    in_place(c)
    c.check("in place", True)


@pytest.mark.parametrize("f16,lens,heads,dk,dv", [(1, [720] * 10, 12, 128, 128), (1, [2000, 1100, 2000], 12, 128, 128),
                                                  (1, [4096, 3600, 4096], 12, 128, 128), (1, [700] * 20, 12, 64, 64),
                                                  (0, [500, 330, 257, 500, 129, 500, 500, 400], 16, 64, 97),
                                                  (0, [900, 260, 900], 24, 128, 64)], ids=str)
def test_in_place_many_blocks(hip, f16, lens, heads, dk, dv):
    """More blocks than run at once, with last pieces of a few rows: states in place give the very bits that states apart
    give, outputs and states."""
    say(f"la in place many {lens} heads {heads} f16 {f16}")
    c = LaCase(hip, lens, heads, heads, heads, heads, dk, dv, f16, gscale=0.02, seed=1)
    c.run()
    want, state = c.do.get(), c.ds1.numpy()
    got, over = in_place(c)
    assert np.isfinite(want).all() and np.array_equal(got, want) and np.array_equal(over, state)


def test_archive_of_some_stations(hip):
    """An hour of 10 stations through the context net at once, and the same rows in calls that are one piece each."""
    from bnneon import contextnet
    net = contextnet.ContextNet(layers=1, stations=10, seed=2)
    rng = np.random.default_rng(3)
    n, step = 720, 240
    x = rng.standard_normal((10, n, net.dim)).astype(np.float32)
    whole = net.plan([n] * 10, range(10))
    assert hip.lib().bnh_linattn_work_bytes(whole["la"][0], n, 10) > 0, "one piece only"
    whole["x"].upload(x.reshape(-1, net.dim))
    say("context net, whole")
    net.run(whole)
    hip.sync()
    got, state = whole["x"].numpy().reshape(x.shape), net.state[0].numpy()
    net.reset()
    part = net.plan([step] * 10, range(10))
    assert hip.lib().bnh_linattn_work_bytes(part["la"][0], step, 10) == 0
    say("context net, in parts")
    for at in range(0, n, step):
        part["x"].upload(np.ascontiguousarray(x[:, at:at + step]).reshape(-1, net.dim))
        net.run(part)
        hip.sync()
        want = part["x"].numpy().reshape(10, step, net.dim)
        # each side's own rounding of a block's rows to fp16, a few parts in 2^11
        off = np.linalg.norm(got[:, at:at + step] - want, axis=(1, 2)) / np.linalg.norm(want, axis=(1, 2))
        say(f"  rows from {at}: {off.max():.2e}")
        assert off.max() < 8 * R.HU
    want = net.state[0].numpy()
    off = np.linalg.norm(state - want) / np.linalg.norm(want)
    say(f"  states: {off:.2e}")
    assert off < 8 * R.HU
