"""Linear attention: a row whose decay e^g is 0 starts the state anew whatever came before it, infinities and NaNs among it."""
import numpy as np
import pytest

import context_ref as R
from test_gpu_context import LaCase, near, say

pytestmark = pytest.mark.gpu
HU = R.HU


def spoil(c, s, at, where, bad):
    """A value that is not finite before row s + at, in head 1."""
    d = c.dk
    row = s + max(0, at - 2)
    if where == "s0":
        c.s0[0, 1, 3, 5] = bad
    elif where == "g":
        c.g[row, 1] = np.nan
    else:
        c.qkv[row, {"q": d + 3, "k": c.hq * d + d + 3, "v": (c.hq + c.hk) * d + c.dv + 3}[where]] = bad


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T,at", [(1, 0), (5, 3), (8, 7), (40, 20), (64, 63), (64, 32), (150, 64), (150, 100), (700, 2),
                                  (700, 299), (700, 640)])
@pytest.mark.parametrize("where", ["s0", "q", "k", "v", "g"])
def test_reset_after_nonfinite(hip, f16, T, at, where):
    """From the reset on, outputs and state are those of a sequence that begins there; the other heads see none of it."""
    if at == 0 and where != "s0":
        pytest.skip("no row before the reset")
    for bad in (np.nan, np.inf):
        for g in (-np.inf, -3.4e38):
            def edit(c):
                spoil(c, 0, at, where, bad)
                c.g[at, 1] = g

            say(f"la reset T {T} at {at} {where} {bad} g {g} f16 {f16}")
            c = LaCase(hip, [T], 3, 3, 3, 3, 32, 48, f16, gscale=0.1, seed=T + at, edit=edit)
            c.run()
            o, s1 = c.do.get()[0].reshape(c.rows, 3, 48), c.ds1.numpy()
            q, k, v = np.split(c.qkv[:T].astype(np.float64), [96, 192], 1)
            q, k, v = q.reshape(T, 3, 32), k.reshape(T, 3, 32), v.reshape(T, 3, 48)
            for h, first in ((0, 0), (1, at), (2, 0)):
                s0 = np.zeros((1, 32, 48)) if h == 1 else c.s0[0, h:h + 1]
                z = slice(first, T)
                wo, ws, eo, es, mo = R.linattn(q[z, h:h + 1], k[z, h:h + 1], v[z, h:h + 1], c.g[z, h:h + 1], c.scale, s0)
                if f16:
                    eo = eo + 3 * HU * mo + 2.0 ** -20 * mo.max(-1, keepdims=True)
                near(o[z, h], wo[:, 0], eo[:, 0], f"head {h} o", f16)
                near(s1[0, h], ws[0], es[0], f"head {h} s")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T", [6, 130, 600])
def test_no_reset_keeps_nonfinite(hip, f16, T):
    """Decays that are small without being 0 keep a state that is not finite so, and a reset in one sequence or head leaves
    the others their own."""
    def edit(c):
        c.s0[:, 1, 3, 5] = np.inf
        c.s0[:, 0, 2, 7] = np.nan
        c.g[:, :] = -3
        c.g[T // 2, 2] = -np.inf
        c.g[c.start[1] + T // 2, 1] = -np.inf

    say(f"la kept T {T} f16 {f16}")
    c = LaCase(hip, [T, T], 3, 3, 3, 3, 32, 48, f16, seed=T, edit=edit)
    c.run()
    s1 = c.ds1.numpy()
    assert not np.isfinite(s1[0, 1, 3, 5]) and not np.isfinite(s1[:, 0, 2, 7]).any()
    assert np.isfinite(s1[1, 1]).all() and np.isfinite(s1[:, 2]).all()


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T,at", [(6, 3), (64, 32), (150, 64), (150, 100), (700, 299)])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_small_values_after_nonfinite(hip, f16, T, at, bad):
    """An infinity that a reset has cleared leaves the small values after it their precision."""
    def edit(c):
        d = slice((c.hq + c.hk) * c.dk, None)
        c.qkv[:, d] = (c.qkv[:, d].astype(np.float32) * 2e-4).astype(c.qkv.dtype)
        c.qkv[at - 2, d] = bad
        c.g[at] = -np.inf

    say(f"la small after {bad} T {T} at {at} f16 {f16}")
    c = LaCase(hip, [T], 2, 2, 2, 2, 32, 48, f16, gscale=0.1, seed=T + at, edit=edit)
    c.run()
    o, s1 = c.do.get()[0].reshape(c.rows, 2, 48)[at:T], c.ds1.numpy()
    q, k, v = (z.reshape(-1, 2, d) for z, d in zip(np.split(c.qkv[at:T].astype(np.float64), [64, 128], 1), (32, 32, 48)))
    wo, ws, eo, es, mo = R.linattn(q, k, v, c.g[at:T], c.scale, np.zeros((2, 32, 48)))
    if f16:
        eo = eo + 3 * HU * mo + 2.0 ** -20 * mo.max(-1, keepdims=True)
    near(o, wo, eo, "o", f16)
    near(s1[0], ws, es, "s")
