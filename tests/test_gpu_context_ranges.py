"""Linear attention over fp16 rows whose values, decays and states are far apart in size."""
import numpy as np
import pytest

from test_gpu_context import LaCase, near, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T,at", [(64, 1), (64, 40), (64, 63), (200, 66), (700, 600)])
@pytest.mark.parametrize("g", [-40.0, -np.inf])
@pytest.mark.parametrize("before,after", [(1e3, 1e-3), (1e4, 1e-3), (6e4, 1e-4)])
def test_large_values_decayed(hip, f16, T, at, g, before, after):
    """A v that a decay takes away within its chunk does not coarsen the state of what comes after."""
    def edit(c):
        v = slice((c.hq + c.hk) * c.dk, None)
        # to a sixth of `before` and of `after`
        for rows, size in ((slice(0, at), before), (slice(at, T), after)):
            c.qkv[rows, v] = (np.clip(c.qkv[rows, v].astype(np.float32), -6, 6) * (size / 6)).astype(c.qkv.dtype)
        c.g[at] = g

    say(f"la decayed T {T} at {at} g {g} {before} {after} f16 {f16}")
    c = LaCase(hip, [T], 2, 2, 2, 2, 64, 48, f16, gscale=0.01, s0=False, seed=T + at, edit=edit)
    c.scale = 1e-3
    c.run()
    c.check("decayed")

@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T", [3, 64, 200, 700])
@pytest.mark.parametrize("state,v", [(1e30, 1e-7), (1e36, 1e-3), (1e-30, 1e4)])
def test_state_of_another_size(hip, f16, T, state, v):
    """A state far larger or smaller than what the rows add to it keeps its own size and precision."""
    def edit(c):
        c.s0 *= np.float32(state)
        d = slice((c.hq + c.hk) * c.dk, None)
        c.qkv[:, d] = (c.qkv[:, d].astype(np.float32) * v).astype(c.qkv.dtype)
        c.scale = 0.1 / max(state, 1.0)

    say(f"la state {state} v {v} T {T} f16 {f16}")
    c = LaCase(hip, [T], 2, 2, 2, 2, 64, 48, f16, gscale=1e-3, seed=T, edit=edit)
    c.run()
    c.check("state")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T", [130, 300])
def test_decayed_state_alone(hip, f16, T):
    """Outputs of a state that has decayed to 2^-58 with no v since, which the caller's scale brings back into range (those
    before are infinite in fp16)."""
    def edit(c):
        c.qkv[:, (c.hq + c.hk) * c.dk:] = 0
        c.g[:] = -1e-3
        c.g[20] = -40.0
        c.scale = 1e17

    say(f"la decayed state T {T} f16 {f16}")
    c = LaCase(hip, [T], 2, 2, 2, 2, 64, 48, f16, seed=T, edit=edit)
    c.run()
    c.check("decayed state")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T", [20, 130])
def test_small_scores(hip, f16, T):
    """Scores below 2^-38 of queries and keys of 1e-6, with large values and a scale to match."""
    def edit(c):
        d = (c.hq + c.hk) * c.dk
        c.qkv[:, :d] = (np.sign(c.qkv[:, :d].astype(np.float32)) * 9.5e-7).astype(c.qkv.dtype)
        c.scale = 1e9

    say(f"la small scores T {T} f16 {f16}")
    c = LaCase(hip, [T], 2, 2, 2, 2, 16, 48, f16, gscale=0.1, s0=False, seed=T, edit=edit)
    c.run()
    c.check("small scores")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("lens,heads,dk,dv", [([64, 9, 200], 4, 128, 128), ([700], 3, 64, 48), ([300, 40], 2, 256, 200),
                                              ([130], 2, 24, 97)], ids=str)
def test_factors_of_22_bits(hip, f16, lens, heads, dk, dv):
    """Outputs whose terms cancel are those of sums in 32 bits of factors of 22 bits (two parts of 11, each of scores and state),
    not of factors of the rows' own type."""
    say(f"la factors lens {lens} dk {dk} dv {dv} f16 {f16}")
    c = LaCase(hip, lens, heads, heads, heads, heads, dk, dv, f16, gscale=0.05, seed=dk)
    c.run()
    o = c.do.get()[0]
    for i in range(len(lens)):
        (wo, _, eo, _, mo), _ = c.want(i)
        s, n = c.sequence(i)
        if f16:  # and of the smallest step of a part beside the largest of its row or column, 2^-37
            eo = eo + 3 * 2.0 ** -22 * mo + 2.0 ** -34 * mo.max(-1, keepdims=True)
        near(o[s:s + n], wo.reshape(n, heads * dv), eo.reshape(n, heads * dv), f"o[{i}]", f16)
