"""Adapters whose first product lies outside fp16's range, or far from the size of its row's others."""
import numpy as np
import pytest

import context_ref as R
from test_gpu_context import LoraCase, near, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,B", [(1, 5), (1, 40), (3, 30), (70, 4), (300, 3)])
@pytest.mark.parametrize("K,N,r", [(64, 136, 16), (1030, 301, 12), (264, 200, 40), (96, 64, 130)])
@pytest.mark.parametrize("size", [1e6, 1e-7])
def test_first_product_out_of_range(hip, M, B, K, N, r, size):
    """a x of 1e6 (past 65504) beside b of 1e-6, and of 1e-7 (below fp16's normal numbers) beside a large scale: outputs are those
    of the definition, to the roundings of the projection's own."""
    def edit(c):
        big = c.a.astype(np.float32) * np.float32(8 if size > 1 else 2.0 ** -6)
        c.a = big.astype(np.float16)
        c.scale = np.full(c.n, size / 8 if size > 1 else size * 64, np.float32)
        c.b = (c.b.astype(np.float32) * (1e-6 if size > 1 else 1000)).astype(np.float16)
        if size < 1:
            c.w[:] = 0
            c.bias[:] = 0

    say(f"lora first product M {M} B {B} K {K} N {N} r {r} {size}")
    c = LoraCase(hip, B, M, N, K, r, 4, seed=M + K, edit=edit)
    got, want, err = c.run(), *R.lora(c.x, c.w, c.bias, c.a, c.b, c.scale, c.idx, c.act, c.res)
    for i, j in enumerate(c.idx):  # the smallest steps of fp16 are those of the row's largest, not of 1
        if j >= 0:
            t = np.abs(c.scale[j] * (c.x[i].astype(np.float64) @ c.a[j].astype(np.float64).T)).max(-1, keepdims=True)
            err[i] += 1.1 * (t * 2.0 ** -39 - R.TINY) * np.abs(c.b[j].astype(np.float64)).sum(-1)
    assert np.isfinite(got).all() and (err >= 0).all()
    near(got, want, err, "first product", True)


@pytest.mark.parametrize("M,B", [(1, 5), (70, 4)])
def test_first_product_not_finite(hip, M, B):
    """An infinity or a NaN among a row's ranks reaches that row alone."""
    def edit(c):
        c.x[1, 0, 3] = np.inf
        c.x[2, M - 1, 5] = np.nan
        c.scale[1] = np.inf

    say(f"lora first product not finite M {M}")
    c = LoraCase(hip, B, M, 136, 64, 16, 4, seed=3, edit=edit, idx=[0, 0, 2, 1, -1][:B])
    with np.errstate(all="ignore"):
        want, err = R.lora(c.x, c.w, c.bias, c.a, c.b, c.scale, c.idx, c.act, c.res)
    got = c.run()
    fine = np.isfinite(want)
    assert not fine.all() and not np.isfinite(got[~fine]).any()
    near(got[fine], want[fine], err[fine], "finite", True)


@pytest.mark.parametrize("M,B", [(1, 7), (1, 60), (5, 30), (90, 3)])
@pytest.mark.parametrize("r", [1, 7, 8, 16, 17, 24, 32, 40, 64, 100, 256])
def test_first_product_of_22_bits(hip, M, B, r):
    """The adapters' part alone, whose terms cancel: as from a first product of 22 bits, not of the rows' own type."""
    def edit(c):
        c.w[:] = 0

    say(f"lora first product of 22 bits M {M} B {B} r {r}")
    c = LoraCase(hip, B, M, 136, 264, r, 5, bias=False, seed=r, edit=edit)
    want, err = R.lora(c.x, c.w, c.bias, c.a, c.b, c.scale, c.idx, c.act, c.res)
    for i, j in enumerate(c.idx):
        if j >= 0:
            t = np.abs(c.scale[j] * (c.x[i].astype(np.float64) @ c.a[j].astype(np.float64).T))
            lost = (R.HU - 2.0 ** -22) * t + R.TINY - t.max(-1, keepdims=True) * 2.0 ** -38
            err[i] -= 1.1 * lost @ np.abs(c.b[j].astype(np.float64)).T
    assert (err >= 0).all()
    near(c.run(), want, err, "22 bits", True)
