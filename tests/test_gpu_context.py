"""The temporal context operators (bnh_block_norm, bnh_pw_lora, bnh_linattn) against their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

import context_ref as R

pytestmark = pytest.mark.gpu
U, HU, TINY = R.U, R.HU, R.TINY


def say(*a):
    print(*a, flush=True)


def near(got, want, err, what, half=False):
    """|got - want| within err, and a rounding to fp16 where the output is; infinities and NaNs in the same places."""
    got, want = got.astype(np.float64), np.asarray(want, np.float64)
    err = np.broadcast_to(np.asarray(err, np.float64), want.shape)
    if half:
        err = err + HU * (np.abs(want) + err) + TINY
    fine = np.isfinite(want)
    if half:
        fine &= np.abs(want) + err < 65504
        big = np.isfinite(want) & (np.abs(want) - err > 65520)
        assert not np.isfinite(got[big]).any(), what
        fine_or_edge = fine | big | ~np.isfinite(want)
    else:
        fine_or_edge = np.ones(want.shape, bool)
    assert np.array_equal(np.isnan(got)[fine_or_edge], np.isnan(want)[fine_or_edge]), what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), what
    assert np.isfinite(got[fine]).all(), what
    off = np.abs(got - want)[fine] / (err[fine] + 1e-300)
    if off.size:
        say(f"  {what}: {off.max():.3f} of the bound")
        assert off.max() <= 1, (what, off.max())


class Rows:
    """A device buffer of B windows of M rows of C values with a row stride, `at` elements into its allocation, the
    space around them filled with a mark."""

    def __init__(self, H, B, M, C, dtype, ld=None, gap=0, at=0, data=None):
        self.H, self.B, self.M, self.C, self.ld = H, B, M, C, C if ld is None else ld
        self.ws = M * self.ld + gap
        self.at, self.dtype = at, np.dtype(dtype)
        host = np.full(at + B * self.ws + 64, 7, self.dtype)
        if data is not None:
            self.view(host)[:] = data
        self.d = H.DeviceArray.from_host(host)
        self.ptr = self.d.ptr + at * self.dtype.itemsize

    def view(self, host):
        body = host[self.at:self.at + self.B * self.ws].reshape(self.B, self.ws)[:, :self.M * self.ld]
        return np.lib.stride_tricks.as_strided(
            body, (self.B, self.M, self.C), (self.ws * self.dtype.itemsize, self.ld * self.dtype.itemsize,
                                             self.dtype.itemsize))

    def get(self):
        host = self.d.numpy()
        out = self.view(host).copy()
        self.view(host)[:] = 7
        assert (host == 7).all(), "written outside the rows"
        return out


# ------------------------------------------------------------------------------------------------ norms
def dev(H, a):
    return None if a is None else H.DeviceArray.from_host(np.asarray(a, np.float32))


class NormCase:
    def __init__(self, H, B, M, C, f16=1, x16=0, post=1, pre=1, gate="rows", gact=1, scale=True, rs=0.5, x=True, f=True,
                 affine=True, pad=0, gap=0, at=0, seed=0, eps=1e-5, mean=0.5, edit=None):
        rng = np.random.default_rng(seed)
        self.H, self.B, self.M, self.C = H, B, M, C
        tf, tx = (np.float16 if f16 else np.float32), (np.float16 if x16 else np.float32)
        self.f16, self.x16, self.gact, self.rs = f16, x16, gact, rs

        def rnd(*s):
            return rng.standard_normal(s).astype(np.float32)

        self.f = (rnd(B, M, C) + mean).astype(tf) if f else None
        self.x = (rnd(B, M, C) * 2).astype(tx) if x else None
        self.gate = None if gate is None else rnd(B, M if gate == "rows" else 1, C).astype(tf)
        self.scale = np.abs(rnd(C)) if scale else None
        self.post = (post, eps, rnd(C) if affine and post else None, rnd(C) if affine and post == 2 else None)
        self.pre = (pre, eps, rnd(C) if affine and pre else None, rnd(C) if affine and pre else None)
        if edit:
            edit(self)
        ld = C + pad

        def rows(a, t, m=M):
            return None if a is None else Rows(H, B, m, C, t, ld, gap, at, a)

        self.df, self.dx = rows(self.f, tf), rows(self.x, tx)
        self.dg = None if gate is None else rows(self.gate, tf, self.gate.shape[1])
        self.dy, self.dn = Rows(H, B, M, C, tx, ld, gap, at), Rows(H, B, M, C, tf, ld, gap, at)
        self.keep = [dev(H, self.scale)] + [dev(H, a) for a in self.post[2:] + self.pre[2:]]

    def args(self):
        H, p = self.H, (lambda d: None if d is None else d.ptr)
        k = [p(d) for d in self.keep]
        a = H.BlockNorm(f16=self.f16, x16=self.x16, gate_act=self.gact, scale=k[0], rs=self.rs,
                        post=H.Norm(self.post[0], self.post[1], k[1], k[2]),
                        pre=H.Norm(self.pre[0], self.pre[1], k[3], k[4]))
        if self.df:
            a.f, a.f_ws, a.ldf = self.df.ptr, self.df.ws, self.df.ld
        if self.dx:
            a.x, a.x_ws, a.ldx = self.dx.ptr, self.dx.ws, self.dx.ld
        if self.dg:
            a.gate, a.g_ws, a.ldg = self.dg.ptr, self.dg.ws, 0 if self.dg.M != self.M else self.dg.ld
            if self.M == 1:
                a.ldg = self.dg.ld
        a.y, a.y_ws, a.ldy = self.dy.ptr, self.dy.ws, self.dy.ld
        a.n, a.n_ws, a.ldn = self.dn.ptr, self.dn.ws, self.dn.ld
        return a

    def run(self, a=None, stream=None):
        H = self.H
        H.check(H.lib().bnh_block_norm(a or self.args(), self.M, self.C, self.B, stream), "block_norm")
        H.sync(stream)

    def check(self, what, y=True, n=True):
        wy, ey, wn, en = R.block_norm(self.f, self.post, self.gate, self.gact, self.scale, self.rs, self.x, self.pre)
        if y:
            near(self.dy.get(), wy, ey, what + " y", self.x16)
        if n:
            near(self.dn.get(), wn, en, what + " n", self.f16)


@pytest.mark.parametrize("f16,x16", [(0, 0), (1, 0), (1, 1)])
@pytest.mark.parametrize("C", [1, 7, 64, 511, 512, 520, 1027, 1536, 2048, 2049, 4104, 8193, 16384])
def test_norm_widths(hip, f16, x16, C):
    say(f"norm C {C} f16 {f16} x16 {x16}")
    c = NormCase(hip, 2, 3, C, f16, x16, post=1, pre=2, seed=C)
    c.run()
    c.check(f"C {C}")


@pytest.mark.parametrize("post", [0, 1, 2])
@pytest.mark.parametrize("pre", [0, 1, 2])
@pytest.mark.parametrize("gate,gact", [(None, 0), ("rows", 0), ("rows", 1), ("window", 3), ("window", 2)])
def test_norm_forms(hip, post, pre, gate, gact):
    say(f"norm post {post} pre {pre} gate {gate} {gact}")
    c = NormCase(hip, 3, 5, 200, 1, 0, post, pre, gate, gact, scale=post != 1, affine=pre != 1, seed=3)
    c.run()
    c.check("forms")


@pytest.mark.parametrize("pad,gap,at", [(8, 16, 8), (3, 5, 1), (0, 1, 0), (8, 0, 4)])
@pytest.mark.parametrize("f16", [0, 1])
def test_norm_strides(hip, pad, gap, at, f16):
    say(f"norm pad {pad} gap {gap} at {at} f16 {f16}")
    c = NormCase(hip, 3, 4, 264, f16, 0, 2, 1, pad=pad, gap=gap, at=at, seed=5)
    c.run()
    c.check("strides")


def test_norm_parts(hip):
    """Entry alone, no residual, either output alone, many windows of one row."""
    say("norm parts")
    c = NormCase(hip, 2, 9, 96, f=False, gate=None, scale=False, seed=7)
    c.run()
    c.check("entry")
    c = NormCase(hip, 2, 9, 96, x=False, seed=8)
    c.run()
    c.check("no residual")
    for drop in ("y", "n"):
        c = NormCase(hip, 300, 1, 96, seed=9)
        a = c.args()
        setattr(a, drop, None)
        c.run(a)
        c.check("one output", y=drop != "y", n=drop != "n")
        left = (c.dy if drop == "y" else c.dn).d.numpy()
        assert (left == 7).all()


def test_norm_in_place(hip):
    """y over x, n over f, and n over the gate's rows, as a caller that keeps one buffer of each has them."""
    for over in ("f", "gate"):
        for C in (96, 1000, 2100):
            say(f"norm in place over x and {over}, C {C}")
            c = NormCase(hip, 2, 17, C, 1, 0, 2, 1, seed=10)
            c.dy, c.dn = c.dx, c.df if over == "f" else c.dg
            c.run()
            c.check("in place")


def test_norm_special_values(hip):
    """A row of zeros, of one value, of huge and of tiny values, an infinity and a NaN in one row and in one gate."""
    def edit(c):
        c.f[0, 0] = 0
        c.f[0, 1] = 3
        c.f[0, 2] *= 6000 / np.abs(c.f[0, 2].astype(np.float32)).max()
        c.f[0, 3] = (c.f[0, 3].astype(np.float32) * 1e-6).astype(c.f.dtype)
        c.f[0, 4, 5] = np.nan
        c.f[0, 5, 5] = np.inf
        c.gate[0, 6, 3] = np.nan
        c.gate[0, 7, 3] = -60000

    for f16 in (0, 1):
        for post in (1, 2):
            say(f"norm special f16 {f16} post {post}")
            c = NormCase(hip, 1, 9, 136, f16, 0, post, 1, seed=11, edit=edit, eps=1e-3)
            c.run()
            with np.errstate(all="ignore"):
                wy, ey, wn, en = R.block_norm(c.f, c.post, c.gate, c.gact, c.scale, c.rs, c.x, c.pre)
            y, n = c.dy.get(), c.dn.get()
            ok = [0, 1, 2, 3, 7, 8]
            near(y[0, ok], wy[0, ok], ey[0, ok], "special y")
            near(n[0, ok], wn[0, ok], en[0, ok], "special n", f16)
            assert np.isnan(y[0, 4]).all() and np.isnan(n[0, 4]).all()
            assert np.isnan(y[0, 5, 5]) and np.isnan(n[0, 5]).all()
            assert np.isnan(y[0, 6, 3]) and np.isfinite(np.delete(y[0, 6], 3)).all() and np.isnan(n[0, 6]).all()


def test_norm_far_rows(hip):
    """Rows past 2^31 elements into their buffer."""
    H = hip
    ld, M, C = 1 << 26, 34, 40
    say("norm far rows")
    rng = np.random.default_rng(12)
    x = rng.standard_normal((M, C)).astype(np.float16)
    big, out = H.DeviceArray((M * ld,), np.float16), H.DeviceArray.zeros((M, C), np.float16)
    for m in range(M):
        H.check(H.lib().bnh_memcpy_h2d(big.ptr + 2 * m * ld, x[m].ctypes.data, 2 * C))
    a = H.BlockNorm(f16=1, x16=1, x=big.ptr, ldx=ld, pre=H.Norm(1, 1e-5, None, None), n=out.ptr, ldn=C)
    H.check(H.lib().bnh_block_norm(a, M, C, 1, None))
    H.sync()
    want, err = R.norm(x.astype(np.float64), 1, 1e-5, None, None)
    near(out.numpy(), want, err, "far", True)


def test_norm_on_a_stream(hip):
    H = hip
    say("norm on a stream")
    s = H.lib().bnh_stream_new()
    c = NormCase(hip, 4, 33, 1536, seed=13)
    c.run(stream=s)
    c.check("stream")
    H.check(H.lib().bnh_stream_free(s))


# ------------------------------------------------------------------------------------------------ adapters
class LoraCase:
    def __init__(self, H, B, M, N, K, r, n, act=0, bias=True, res=False, scale=True, idx=None, padx=0, padw=0, pado=0,
                 gap=0, at=0, seed=0, edit=None):
        rng = np.random.default_rng(seed)
        self.H, self.B, self.M, self.N, self.K, self.r, self.n, self.act = H, B, M, N, K, r, n, act

        def rnd(*s, std=1.0):
            return (rng.standard_normal(s) * std).astype(np.float32)

        self.x = rnd(B, M, K).astype(np.float16)
        self.w = rnd(N, K, std=K ** -0.5).astype(np.float16)
        self.bias = rnd(N) if bias else None
        self.a = rnd(n, r, K, std=K ** -0.5).astype(np.float16) if n else None
        self.b = rnd(n, N, r, std=r ** -0.5).astype(np.float16) if n else None
        self.scale = rng.uniform(0.5, 2, n).astype(np.float32) if scale and n else None
        self.res = rnd(B, M, N).astype(np.float16) if res else None
        self.idx = np.asarray(rng.integers(-1, n, B) if idx is None else idx, np.int32) if n else np.full(B, -1)
        if edit:
            edit(self)
        self.dx = Rows(H, B, M, K, np.float16, K + padx, gap, at, self.x)
        self.dw = Rows(H, 1, N, K, np.float16, K + padw, 0, at, self.w)
        self.do = Rows(H, B, M, N, np.float16, N + pado, gap, at)
        self.dr = Rows(H, B, M, N, np.float16, N + pado, gap, at, self.res) if res else None
        self.da, self.db = (Rows(H, 1, 1, z.size, np.float16, None, 0, at, z.ravel()) if n else None
                            for z in (self.a, self.b))
        self.dbias, self.dscale = dev(H, self.bias), dev(H, self.scale)
        self.didx = H.DeviceArray.from_host(self.idx.astype(np.int32))

    def run(self, stream=None, out=None):
        H, p = self.H, (lambda d: None if d is None else d.ptr)
        L = H.lib()
        wb = L.bnh_pw_lora_work_bytes(self.M, self.B, self.N, self.K, self.r)
        ws = H.DeviceArray.from_host(np.full(wb + 256, 0xff, np.uint8))  # NaNs where nothing is written
        ad = H.Lora(self.n, self.r, p(self.da), p(self.db), p(self.dscale)) if self.n else None
        o = out or self.do
        e = H.Epi16(self.act, o.ptr, o.ws, o.ld, 0, 0, p(self.dr), self.dr.ws if self.dr else 0,
                    self.dr.ld if self.dr else 0)
        H.check(L.bnh_pw_lora(self.dx.ptr, self.dx.ws, self.dx.ld, self.M, self.B, self.dw.ptr, self.dw.ld, self.N,
                              self.K, p(self.dbias), ad, self.didx.ptr, e, ws.ptr, wb, stream), "pw_lora")
        H.sync(stream)
        assert (ws.numpy()[wb:] == 0xff).all(), "written past the workspace"
        return o.get()

    def check(self, what, got=None):
        want, err = R.lora(self.x, self.w, self.bias, self.a, self.b, self.scale, self.idx, self.act, self.res)
        near(self.run() if got is None else got, want, err, what, True)


@pytest.mark.parametrize("M,B", [(1, 1), (1, 3), (1, 16), (1, 33), (2, 20), (5, 13), (64, 2), (65, 3), (200, 2), (300, 4)])
@pytest.mark.parametrize("K,N,r", [(64, 128, 16), (200, 136, 8), (129, 61, 5), (1030, 301, 12)])
def test_lora_rows(hip, M, B, K, N, r):
    say(f"lora M {M} B {B} K {K} N {N} r {r}")
    LoraCase(hip, B, M, N, K, r, 7, act=M % 3, res=M % 2 == 1, seed=M + K).check("rows")


@pytest.mark.parametrize("r", [1, 8, 16, 24, 32, 33, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("M,B", [(1, 20), (40, 5)])
def test_lora_ranks(hip, r, M, B):
    say(f"lora rank {r} M {M}")
    LoraCase(hip, B, M, 144, 96, r, 4, seed=r).check("rank")


@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (31, 17), (40, 1000), (1536, 128), (1536, 1536), (2050, 40)])
@pytest.mark.parametrize("M", [1, 30, 260])
def test_lora_shapes(hip, K, N, M):
    say(f"lora K {K} N {N} M {M}")
    LoraCase(hip, 2, M, N, K, 16, 3, seed=K + N).check("shape")


@pytest.mark.parametrize("padx,padw,pado,gap,at", [(8, 16, 24, 32, 8), (1, 3, 5, 7, 1), (2, 2, 2, 2, 2), (0, 0, 1, 0, 0),
                                                   (8, 8, 8, 3, 4)])
@pytest.mark.parametrize("M", [1, 70])
def test_lora_strides(hip, padx, padw, pado, gap, at, M):
    say(f"lora strides {padx} {padw} {pado} {gap} {at} M {M}")
    LoraCase(hip, 5, M, 200, 264, 16, 3, act=1, res=True, padx=padx, padw=padw, pado=pado, gap=gap, at=at,
             seed=M).check("strides")


@pytest.mark.parametrize("M", [1, 3, 50])
def test_lora_ids(hip, M):
    """Every window its own, all the same, none, ids outside the list, no scale, no bias, no adapters at all."""
    B = 40
    for name, idx in (("own", np.arange(B)), ("same", np.full(B, 5)), ("none", np.full(B, -1)),
                      ("outside", np.where(np.arange(B) % 3 == 0, 1000, np.arange(B) % 5 - 2)),
                      ("runs", np.arange(B) // 9)):
        say(f"lora ids {name} M {M}")
        LoraCase(hip, B, M, 136, 72, 8, B, idx=idx, scale=name != "runs", bias=name != "own", seed=2).check(name)
    LoraCase(hip, B, M, 136, 72, 8, 0, seed=2).check("no adapters")


@pytest.mark.parametrize("M", [1, 4, 33])
def test_lora_requests_apart(hip, M):
    """Non-finite values of one station's adapter and rows stay with that station's rows, and unwritten workspace too."""
    def edit(c):
        c.a[1, 2, 3] = np.nan
        c.b[2, 5, 1] = np.inf
        c.b[3] = np.nan
        c.x[4, 0, 7] = np.inf
        c.x[9, 0, 2] = np.nan

    idx = np.array([0, 1, 2, 3, 0, -1, 0, 1, 0, -1, 2, 0])
    c = LoraCase(hip, 12, M, 72, 64, 8, 4, idx=idx, seed=4, edit=edit)
    say(f"lora apart M {M}")
    with np.errstate(all="ignore"):
        want, err = R.lora(c.x, c.w, c.bias, c.a, c.b, c.scale, c.idx, c.act, c.res)
    got = c.run()
    fine = np.isfinite(want)
    assert np.isfinite(got[fine]).all()
    near(got[fine], want[fine], err[fine], "apart", True)
    assert not np.isfinite(got[~fine]).any()


@pytest.mark.parametrize("M,B,N,K,r", [(41, 101, 3080, 136, 16), (1, 4100, 3080, 40, 24), (700, 6, 3080, 64, 40),
                                       (41, 51, 2048, 136, 16), (41, 51, 2048, 200, 12), (41, 51, 2049, 130, 12),
                                       (1, 2080, 2048, 130, 33), (700, 3, 2056, 32, 8)])
def test_lora_large_tiles(hip, M, B, N, K, r):
    """Outputs enough for each of the larger tiles, whole and ragged, with rows of several adapters in a tile, one of them
    not finite."""
    def edit(c):
        c.b[2, N // 3, 1] = np.nan

    say(f"lora large M {M} B {B} N {N} K {K} r {r}")
    c = LoraCase(hip, B, M, N, K, r, 9, act=M % 3 % 2, res=M == 41, seed=N + K, edit=edit, idx=(np.arange(B) + 2) % 10)
    with np.errstate(all="ignore"):
        want, err = R.lora(c.x, c.w, c.bias, c.a, c.b, c.scale, c.idx, c.act, c.res)
    got = c.run()
    fine = np.isfinite(want)
    assert not fine.all() and not np.isfinite(got[~fine]).any()
    near(got[fine], want[fine], err[fine], "large", True)


def test_lora_residual_in_place(hip):
    for M, N in ((1, 136), (70, 136), (70, 61)):
        say(f"lora in place M {M} N {N}")
        c = LoraCase(hip, 6, M, N, 72, 8, 4, act=2, res=True, seed=6)
        c.check("in place", c.run(out=c.dr))


def test_lora_far_rows(hip):
    """Rows of x and out past 2^31 elements into their buffers."""
    H = hip
    M, K, N, ld = 34, 64, 64, 1 << 26
    say("lora far rows")
    c = LoraCase(hip, 1, M, N, K, 8, 2, idx=[1], seed=14)
    big, out = H.DeviceArray((M * ld,), np.float16), H.DeviceArray((M * ld,), np.float16)
    for m in range(M):
        H.check(H.lib().bnh_memcpy_h2d(big.ptr + 2 * m * ld, c.x[0, m].ctypes.data, 2 * K))
    L = H.lib()
    wb = L.bnh_pw_lora_work_bytes(M, 1, N, K, 8)
    ws = H.DeviceArray((wb,), np.uint8)
    ad = H.Lora(2, 8, c.da.ptr, c.db.ptr, c.dscale.ptr)
    H.check(L.bnh_pw_lora(big.ptr, 0, ld, M, 1, c.dw.ptr, K, N, K, c.dbias.ptr, ad, c.didx.ptr,
                          H.Epi16(0, out.ptr, 0, ld, 0, 0, None, 0, 0), ws.ptr, wb, None))
    H.sync()
    got = np.empty((1, M, N), np.float16)
    for m in range(M):
        H.check(L.bnh_memcpy_d2h(got[0, m].ctypes.data, out.ptr + 2 * m * ld, 2 * N))
    c.check("far", got)


# ------------------------------------------------------------------------------------------------ linear attention
class LaCase:
    """Sequences of the given lengths, side by side in one buffer of q, k and v (and `pad` more values a row)."""

    def __init__(self, H, lens, heads, hq, hk, hv, dk, dv, f16, s0=True, s1=True, ldg=True, pad=0, at=0, T=None, seed=0,
                 gap=0, gscale=1.0, std=1.0, edit=None, uniform=False, slot=None, slots=None):
        rng = np.random.default_rng(seed)
        self.H, self.lens, self.heads, self.hq, self.hk, self.hv = H, lens, heads, hq, hk, hv
        self.dk, self.dv, self.f16, self.T = dk, dv, f16, T or max(1, max(lens))
        self.uniform, B = uniform, len(lens)
        t = np.float16 if f16 else np.float32
        self.start = np.cumsum([0] + [n + gap for n in lens[:-1]]).astype(np.int32)
        self.rows = int(self.start[-1] + max(lens[-1], 1) + gap)
        if uniform:
            self.start = (np.arange(B) * self.T).astype(np.int32)
            self.rows = B * self.T
        self.width = hq * dk + hk * dk + hv * dv
        self.qkv = (rng.standard_normal((self.rows, self.width)) * std).astype(t)
        n = self.rows if ldg else 1
        self.g = (-np.abs(rng.standard_normal((n, heads)) * gscale * np.linspace(0.01, 1, heads))).astype(np.float32)
        self.slot = None if slot is None else np.asarray(slot, np.int32)
        self.slots = slots or B
        self.s0 = rng.standard_normal((self.slots, heads, dk, dv)).astype(np.float32) if s0 else None
        self.scale = 0.3
        if edit:
            edit(self)
        self.dqkv = Rows(H, 1, self.rows, self.width, t, self.width + pad, 0, at, self.qkv)
        self.do = Rows(H, 1, self.rows, heads * dv, t, heads * dv + pad, 0, at)
        self.dg = Rows(H, 1, n, heads, np.float32, heads + (3 if ldg else 0), 0, at, self.g)
        self.ds0 = H.DeviceArray.from_host(self.s0) if s0 else None
        self.ds1 = H.DeviceArray.from_host(np.full((self.slots, heads, dk, dv), 7, np.float32)) if s1 else None
        self.dstart, self.dlen = (H.DeviceArray.from_host(np.asarray(z, np.int32)) for z in (self.start, lens))
        self.dslot = None if slot is None else H.DeviceArray.from_host(self.slot)
        self.ldg = self.dg.ld if ldg else 0

    def args(self):
        H, es, p = self.H, 2 if self.f16 else 4, (lambda d: None if d is None else d.ptr)
        q = self.dqkv.ptr
        return H.LinAttn(q=q, k=q + es * self.hq * self.dk, v=q + es * (self.hq + self.hk) * self.dk, o=self.do.ptr,
                         f16=self.f16, ldq=self.dqkv.ld, ldk=self.dqkv.ld, ldv=self.dqkv.ld, ldo=self.do.ld,
                         H=self.heads, Hq=self.hq, Hk=self.hk, Hv=self.hv, dk=self.dk, dv=self.dv, g=self.dg.ptr,
                         ldg=self.ldg, scale=self.scale, s0=p(self.ds0), s1=p(self.ds1), slots=self.slots,
                         slot=p(self.dslot))

    def run(self, stream=None):
        H, L, a = self.H, self.H.lib(), self.args()
        B = len(self.lens)
        wb = L.bnh_linattn_work_bytes(a, self.T, B)
        ws = H.DeviceArray.from_host(np.full(wb + 256, 0xff, np.uint8))
        H.check(L.bnh_linattn(a, self.T, B, self.rows, None if self.uniform else self.dstart.ptr,
                              None if self.uniform else self.dlen.ptr, ws.ptr if wb else None, wb, stream), "linattn")
        H.sync(stream)
        assert (ws.numpy()[wb:] == 0xff).all(), "written past the workspace"

    def sequence(self, i):
        """(first row, rows) as the entry point cuts them"""
        s, n = int(self.start[i]), min(int(self.lens[i]), self.T)
        return (s, max(0, min(n, self.rows - s))) if 0 <= s < self.rows else (0, 0)

    def want(self, i):
        s, n = self.sequence(i)
        dk, dv, h = self.dk, self.dv, self.heads
        x = self.qkv[s:s + n].astype(np.float64)
        q, k, v = np.split(x, [self.hq * dk, (self.hq + self.hk) * dk], 1)
        q, k, v = (np.repeat(z.reshape(n, c, d), h // c, 1)
                   for z, c, d in ((q, self.hq, dk), (k, self.hk, dk), (v, self.hv, dv)))
        g = self.g[s:s + n] if self.ldg else np.repeat(self.g, n, 0)
        j = i if self.slot is None else int(self.slot[i])
        s0 = self.s0[j] if self.s0 is not None and 0 <= j < self.slots else np.zeros((h, dk, dv))
        return R.linattn(q, k, v, g, self.scale, s0), j

    def check(self, what, s0_was_s1=False):
        o = self.do.get()[0]
        s1 = None if self.ds1 is None else self.ds1.numpy()
        seen_rows, seen_slots = np.zeros(self.rows, bool), np.zeros(self.slots, bool)
        for i in range(len(self.lens)):
            (wo, ws, eo, es, mo), j = self.want(i)
            s, n = self.sequence(i)
            seen_rows[s:s + n] = True
            if self.f16:  # the factors of o's products are rounded to fp16, the state's against its largest
                eo = eo + 3 * HU * mo + 2.0 ** -20 * (mo.max(-1, keepdims=True) if mo.size else 0)
            near(o[s:s + n], wo.reshape(n, self.heads * self.dv), eo.reshape(n, self.heads * self.dv), f"{what} o[{i}]", self.f16)
            if s1 is not None and 0 <= j < self.slots:
                seen_slots[j] = True
                near(s1[j], ws, es, f"{what} s[{i}]")
        assert (o[~seen_rows] == 7).all(), "rows of no sequence were written"
        if s1 is not None:
            assert (s1[~seen_slots] == 7).all() or s0_was_s1, "states of no sequence were written"


LENGTHS = [[1], [1, 1, 1], [2, 1, 0, 3], [5, 17], [63], [64], [65], [31, 128, 1, 0, 129], [200], [257, 96], [1000, 3],
           [0], [0, 0, 40]]


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_la_lengths(hip, f16, lens):
    say(f"la lens {lens} f16 {f16}")
    c = LaCase(hip, lens, 4, 2, 4, 4, 64, 48, f16, seed=len(lens))
    c.run()
    c.check("lengths")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (16, 16), (24, 40), (32, 130), (64, 97), (100, 64), (128, 128),
                                   (129, 33), (200, 256), (256, 200), (256, 256)])
@pytest.mark.parametrize("T", [1, 4, 70])
def test_la_dims(hip, f16, dk, dv, T):
    say(f"la dk {dk} dv {dv} T {T} f16 {f16}")
    c = LaCase(hip, [T, max(1, T - 3)], 2, 2, 1, 2, dk, dv, f16, seed=dk + dv)
    c.run()
    c.check("dims")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 128), (128, 128), (100, 77), (256, 136)])
def test_la_pieces(hip, f16, dk, dv):
    """Long sequences in pieces that are joined, ends inside and at the end of pieces, with a short one beside them."""
    say(f"la pieces dk {dk} dv {dv} f16 {f16}")
    c = LaCase(hip, [1024, 700, 5, 0, 513], 2, 2, 2, 2, dk, dv, f16, gscale=0.1, seed=dk)
    c.run()
    c.check("pieces")


@pytest.mark.parametrize("hq,hk,hv", [(12, 12, 12), (1, 1, 12), (6, 3, 4), (2, 12, 1)])
@pytest.mark.parametrize("T", [1, 90])
def test_la_heads(hip, hq, hk, hv, T):
    say(f"la heads {hq} {hk} {hv} T {T}")
    c = LaCase(hip, [T, T, T], 12, hq, hk, hv, 32, 32, 1, uniform=True, ldg=T == 1, s0=T == 1, seed=hq)
    c.run()
    c.check("heads")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("pad,at", [(8, 8), (1, 3), (16, 1)])
@pytest.mark.parametrize("T", [1, 75])
def test_la_strides(hip, f16, pad, at, T):
    say(f"la strides pad {pad} at {at} T {T} f16 {f16}")
    c = LaCase(hip, [T, T // 2 + 1], 3, 3, 3, 3, 64, 64, f16, pad=pad, at=at, gap=2, seed=pad)
    c.run()
    c.check("strides")


@pytest.mark.parametrize("T", [1, 6, 100])
def test_la_slots(hip, T):
    """States of a pool by slot, slots outside it, states in place, no states at all."""
    say(f"la slots T {T}")
    c = LaCase(hip, [T, T, 0, T, 1], 2, 2, 2, 2, 32, 64, 1, slot=[6, 0, 3, -1, 900], slots=8, seed=T)
    c.run()
    c.check("slots")
    c = LaCase(hip, [T, T, 0], 2, 2, 2, 2, 32, 64, 1, slot=[6, 0, 3], slots=8, seed=T)
    c.ds1 = c.ds0
    c.run()
    kept = [i for i in range(8) if i not in (6, 0, 3)]
    assert np.array_equal(c.ds0.numpy()[kept], c.s0[kept])
    c.check("in place", True)
    for s0, s1 in ((False, True), (True, False), (False, False)):
        c = LaCase(hip, [T, T], 2, 2, 2, 2, 32, 64, 0, s0=s0, s1=s1, seed=T)
        c.run()
        c.check(f"s0 {s0} s1 {s1}")


@pytest.mark.parametrize("f16", [0, 1])
def test_la_cut_sequences(hip, f16):
    """Lengths past T, starts and ends past the buffers' rows, a negative start and a negative length."""
    c = LaCase(hip, [80, 80, 80, 80, 30], 2, 2, 2, 2, 32, 32, f16, T=70, seed=1)
    say(f"la cut f16 {f16}")
    c.lens = [80, 500, -4, 80, 80]
    c.start = np.array([0, 80, 160, -5, c.rows - 9], np.int32)
    c.dstart, c.dlen = (hip.DeviceArray.from_host(np.asarray(z, np.int32)) for z in (c.start, c.lens))
    c.run()
    c.check("cut")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_la_decays(hip, f16, T):
    """Decays of 1, resets (-inf) in runs and alone, very small decays, decays that differ by row."""
    def edit(c):
        c.g[:, 0] = 0
        c.g[::7, 1] = -np.inf
        c.g[T // 2:T // 2 + 3, 2] = -np.inf
        c.g[:, 3] = -60
        c.g[::3, 3] = -0.01
        c.g[:, 4] = -1e30
        c.g[1::2, 4] = -1e-3

    say(f"la decays T {T} f16 {f16}")
    c = LaCase(hip, [T, T], 5, 5, 5, 5, 40, 24, f16, seed=T, edit=edit)
    c.run()
    c.check("decays")


@pytest.mark.parametrize("T", [1, 50, 200])
def test_la_large_values(hip, T):
    """fp16 rows whose state and scores are far past the largest fp16 number while the outputs are not."""
    def edit(c):
        c.qkv[:, :64] *= np.float16(0.004)          # q
        c.qkv[:, 64:128] = 40 + 20 * c.qkv[:, 64:128]  # k
        c.qkv[:, 128:] = 30 + 10 * c.qkv[:, 128:]   # v
        c.g[:] = -1e-4
        c.scale = 2e-3

    say(f"la large T {T}")
    c = LaCase(hip, [T], 2, 2, 2, 2, 32, 32, 1, s0=False, seed=T, edit=edit)
    c.run()
    c.check("large")

    def scores(c):
        c.qkv[:, :64] = 50 + 5 * c.qkv[:, :64]
        c.qkv[:, 64:128] = 60 + 5 * c.qkv[:, 64:128]
        c.qkv[:, 128:] *= np.float16(0.01)
        c.scale = 1e-3

    c = LaCase(hip, [T], 2, 2, 2, 2, 32, 32, 1, s0=False, seed=T, edit=scores)
    c.run()
    c.check("large scores")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T", [5, 64, 150])
@pytest.mark.parametrize("where", ["q", "k", "v", "g"])
def test_la_nonfinite_rows(hip, f16, T, where):
    """An infinity and a NaN at one row reach neither the rows before it nor another head or sequence."""
    at = 2 * T // 3
    for bad in (np.nan, np.inf):
        def edit(c):
            row = c.start[0] + at
            if where == "g":
                c.g[row, 1] = np.nan
            else:
                c.qkv[row, {"q": 33, "k": 3 * 32 + 33, "v": 6 * 32 + 33}[where]] = bad

        say(f"la nonfinite {where} {bad} T {T} f16 {f16}")
        c = LaCase(hip, [T, T], 3, 3, 3, 3, 32, 32, f16, seed=T, edit=edit)
        c.run()
        o = c.do.get()[0].astype(np.float64).reshape(c.rows, 3, 32)
        s1 = c.ds1.numpy()
        (wo, ws, eo, es, mo), _ = c.want(0)
        (vo, vs, fo, fs, no), _ = c.want(1)
        if f16:
            fo, eo = fo + 3 * HU * no + 2.0 ** -20 * no.max(-1, keepdims=True), eo + 3 * HU * mo
            eo = eo + 2.0 ** -20 * np.where(np.isfinite(mo), mo, 0).max(-1, keepdims=True)
        s = c.start[1]
        near(o[s:s + T], vo, fo, "other sequence", f16)
        near(s1[1], vs, fs, "other state")
        for h in (0, 2):
            near(o[:T, h], wo[:, h], eo[:, h], f"head {h}", f16)
            near(s1[0, h], ws[h], es[h], f"state {h}")
        near(o[:at, 1], wo[:at, 1], eo[:at, 1], "rows before", f16)
        if where == "q":
            near(o[at + 1:T, 1], wo[at + 1:, 1], eo[at + 1:, 1], "rows after", f16)
            near(s1[0, 1], ws[1], es[1], "state")
            assert not np.isfinite(o[at, 1]).all()
        else:
            bad_o, bad_s = ~np.isfinite(wo[:, 1]), ~np.isfinite(ws[1])
            assert not np.isfinite(o[:T, 1][bad_o]).any() and not np.isfinite(s1[0, 1][bad_s]).any()
            fine = ~bad_o
            near(o[:T, 1][fine], wo[:, 1][fine], eo[:, 1][fine], "finite columns", f16)
            near(s1[0, 1][~bad_s], ws[1][~bad_s], es[1][~bad_s], "finite columns of the state")


def test_la_far_rows(hip):
    """Rows past 2^31 elements into their buffer, for one row a sequence and for a chunk of them."""
    H = hip
    ld, T, d = 1 << 25, 72, 32
    rng = np.random.default_rng(15)
    x = rng.standard_normal((T, 3 * d)).astype(np.float16)
    big = H.DeviceArray((T * ld,), np.float16)
    g, o = H.DeviceArray.from_host(np.full(1, -0.1, np.float32)), H.DeviceArray.zeros((T, d), np.float16)
    for m in range(T):
        H.check(H.lib().bnh_memcpy_h2d(big.ptr + 2 * m * ld, x[m].ctypes.data, 6 * d))
    for n, B in ((T, 1), (1, T)):
        say(f"la far rows T {n}")
        a = H.LinAttn(q=big.ptr, k=big.ptr + 2 * d, v=big.ptr + 4 * d, o=o.ptr, f16=1, ldq=ld, ldk=ld, ldv=ld, ldo=d,
                      H=1, Hq=1, Hk=1, Hv=1, dk=d, dv=d, g=g.ptr, ldg=0, scale=1.0)
        wb = H.lib().bnh_linattn_work_bytes(a, n, B)
        ws = H.DeviceArray((max(1, wb),), np.uint8)
        H.check(H.lib().bnh_linattn(a, n, B, T, None, None, ws.ptr, wb, None))
        H.sync()
        for i in range(B):
            q, k, v = (z[:, None] for z in np.split(x[i * n:(i + 1) * n], 3, 1))
            wo, _, eo, _, mo = R.linattn(q, k, v, np.full((n, 1), -0.1), 1.0, np.zeros((1, d, d)))
            near(o.numpy()[i * n:(i + 1) * n], wo[:, 0], (eo + 3 * HU * mo)[:, 0], "far", True)


def test_la_many_heads_and_sequences(hip):
    """More sequences and heads than the card has compute units, at lengths that both forms take."""
    for T in (1, 33):
        say(f"la many T {T}")
        c = LaCase(hip, [T] * 70, 8, 8, 8, 8, 16, 16, 1, uniform=True, seed=T)
        c.run()
        c.check("many")
