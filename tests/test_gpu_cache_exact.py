"""Cached attention where its precision shows: weights as factors of 22 bits in every form, scales near the smallest, far angles."""
import numpy as np
import pytest

import cache_ref as R
from test_gpu_cache import TWO, Append, Attn
from test_gpu_context import near, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dk,dv", [(16, 16), (64, 64), (64, 128), (128, 64), (128, 128), (256, 256), (200, 72), (127, 127), (126, 98)])
@pytest.mark.parametrize("heads,hk,n", [(1, 1, 16), (1, 1, 17), (2, 1, 20), (3, 3, 40)])
@pytest.mark.parametrize("page", [16, 128])
def test_weights_of_many_rows(hip, dk, dv, heads, hk, n, page):
    """A row's weights are as exact beside many rows as alone. Few tokens and small scores, so that 32-bit sums leave less than
    11 bits would."""
    say(f"weights {dk} {dv} heads {heads} {hk} rows {n} page {page}")
    a = Attn(hip, [0, 9, 30], [n, n, n - 1], heads, hk, dk, dv, page, 1, seed=dk + n, qstd=2.0 / dk ** 0.5)
    a.run()
    a.check("weights", TWO)


@pytest.mark.parametrize("n", [1, 16, 40])
@pytest.mark.parametrize("d", [64, 256])
def test_mean_of_the_largest(hip, d, n):
    """A mean of equal values is that value, also of fp16's largest: 22 bits of a weight are 2^-22 off, half a step is 2^-12."""
    say(f"largest rows {n} d {d}")

    def edit(c):
        for i in range(c.B):
            c.V[i][:] = 65504

    a = Attn(hip, [0, 300], [n, n], 2, 1, d, d, 32, 1, seed=n, edit=edit)
    a.run()
    got = a.do.get()[0].reshape(a.c.rows, -1)
    for s in a.c.start:
        assert (got[s:s + n].astype(np.float32) == 65504).all()


@pytest.mark.parametrize("f16,d,n", [(1, 64, 1), (1, 128, 200), (0, 64, 1), (0, 64, 100)])
def test_a_window_wider_than_any_cache_in_parts(hip, f16, d, n):
    """As no window: the same parts, the same output."""
    say(f"widest window rows {n} d {d} f16 {f16}")
    got = []
    for window in (0, 2 ** 31 - 1):
        a = Attn(hip, [2000, 40], [n, n], 3, 1, d, d, 64, f16, window=window, seed=n)
        assert hip.lib().bnh_kv_attn_work_bytes(a.c.args(), a.args(), *a.c.seqs()[:3]) > 0
        a.run()
        a.check("window")
        got.append(a.do.get()[0].copy())
    assert np.array_equal(*got)


@pytest.mark.parametrize("n", [1, 20, 100])
@pytest.mark.parametrize("scale", [0.0, 5e-39, 2e-38, -6e-38, 2e-37])
def test_small_scales_of_large_scores(hip, scale, n):
    """fp32 products of 1e37 times a scale near fp32's smallest, or of 0: scores are what the two give."""
    say(f"scale {scale} rows {n}")
    scale = float(np.float32(scale))
    a = Attn(hip, [90, 0], [n, n], 4, 2, 64, 64, 32, 0, seed=n, qstd=1e18, std=1e18, scale=scale)
    a.run()
    a.check(f"scale {scale}")


@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("first", [1.0, 0.37, 3e4, 2e6])
def test_far_angles(hip, first, pairs):
    """An angle is as exact at positions of 2^31 as near 0: against cos and sin of products that 64 bits of mantissa hold whole
    (31 + 24 bits), within the bound of 32-bit arithmetic on exact angles."""
    say(f"far angles {first} pairs {pairs}")
    assert np.finfo(np.longdouble).nmant >= 63

    def pos(c):
        p = np.random.default_rng(3).integers(-2 ** 31, 2 ** 31, c.rows)
        p[:5] = 2 ** 31 - 1, -2 ** 31, 0, 1, 2 ** 30 + 1
        return p

    a = Append(hip, [3, 0], [400, 150], 1, 1, 256, 8, 256, pairs, 16, 0, pos=pos, seed=pairs)
    a.freq = (first * np.geomspace(1, 1e-3, 128)).astype(np.float32)
    a.dfreq.upload(a.freq)
    a.run()
    got = a.dqr.get()[0].reshape(a.c.rows, 256).astype(np.float64)
    e = np.arange(128)
    i, j = (2 * e, 2 * e + 1) if pairs else (e, e + 128)
    for s, n in zip(a.c.start, a.c.lens):
        t = a.pos[s:s + n].astype(np.longdouble)[:, None] * a.freq.astype(np.longdouble)
        x, y = (a.q[s:s + n, 0][:, k].astype(np.float64) for k in (i, j))
        cs, sn = np.cos(t).astype(np.float64), np.sin(t).astype(np.float64)
        err = 6 * R.U * (np.abs(x) + np.abs(y))
        near(got[s:s + n][:, i], x * cs - y * sn, err, "x")
        near(got[s:s + n][:, j], x * sn + y * cs, err, "y")
