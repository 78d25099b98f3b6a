"""The cached-attention operators (bnh_kv_append, bnh_kv_attn, bnh_kv_select) against their definitions in 64 bits."""
import numpy as np
import pytest

import cache_ref as R
from test_gpu_context import Rows, near, say

pytestmark = pytest.mark.gpu
U, HU = R.U, R.HU
# what weights are rounded by as factors: two fp16 parts, or one
TWO, ONE = 2.0 ** -21, HU


def typ(f16):
    return np.float16 if f16 else np.float32


class Cache:
    """Sequences of past + new tokens, the first `held` (a number each; default: all) of them in pages of a pool in random
    order; everything else in the pool is `fill`. K[i], V[i]: a sequence's tokens; `gone`: pages (of a sequence, in its order)
    that are not there."""

    def __init__(self, H, pasts, lens, hk, dk, dv, page=32, f16=1, seed=0, held=None, extra=0, fill=np.nan, gone=(), more=1,
                 std=1.0, bounds=True, edit=None, T=None, at=0):
        rng = np.random.default_rng(seed)
        self.H, self.pasts, self.lens, self.hk, self.dk, self.dv, self.page, self.f16 = H, pasts, lens, hk, dk, dv, page, f16
        self.B, self.T, self.t = len(lens), T or max(1, max(lens)), typ(f16)
        self.total = [p + n for p, n in zip(pasts, lens)]
        self.K = [(rng.standard_normal((n, hk, dk)) * std).astype(self.t) for n in self.total]
        self.V = [rng.standard_normal((n, hk, dv)).astype(self.t) for n in self.total]
        need = [-(-n // page) for n in self.total]
        self.pages, self.ldt = sum(need) + 2, max(need) + more
        order = rng.permutation(self.pages)
        self.table = np.full((self.B, self.ldt), -1, np.int32)
        self.table[:, -1] = self.pages + 3
        for i in range(self.B):
            self.table[i, :need[i]] = order[sum(need[:i]):sum(need[:i + 1])]
        for i, x in gone:
            if x < self.ldt:
                self.table[i, x] = -1 if x % 2 else self.pages
        if edit:
            edit(self)
        self.k_ps, self.v_ps, self.at = hk * page * dk + extra, hk * page * dv + extra, at
        self.held = self.total if held is None else held
        self.kb, self.vb = (np.full(at + self.pages * n, fill, self.t) for n in (self.k_ps, self.v_ps))
        self.lo, self.hi = (np.full((self.pages, hk, dk), 3, self.t) for _ in range(2))
        for i in range(self.B):
            self.store(i, 0, self.held[i])
        self.dk_, self.dv_ = H.DeviceArray.from_host(self.kb), H.DeviceArray.from_host(self.vb)
        self.dlo, self.dhi = (H.DeviceArray.from_host(x) if bounds else None for x in (self.lo, self.hi))
        self.dtable, self.dpast = H.DeviceArray.from_host(self.table), H.DeviceArray.from_host(np.array(pasts, np.int32))
        self.start = np.cumsum([0] + [n + 1 for n in lens[:-1]]).astype(np.int32)  # a row of nobody's after each
        self.rows = int(self.start[-1] + lens[-1] + 1)
        self.dstart, self.dlen = H.DeviceArray.from_host(self.start), H.DeviceArray.from_host(np.array(lens, np.int32))

    def place(self, buf, ps, d):
        """[pages][hk][page][d] of a pool's buffer"""
        return buf[self.at:].reshape(self.pages, ps)[:, :self.hk * self.page * d].reshape(self.pages, self.hk, self.page, d)

    def store(self, i, a, b):
        """Tokens [a, b) of sequence i into the host's pool and bounds."""
        kc, vc = self.place(self.kb, self.k_ps, self.dk), self.place(self.vb, self.v_ps, self.dv)
        for j in range(a, b):
            x = self.table[i, j // self.page] if j // self.page < self.ldt else -1
            if 0 <= x < self.pages:
                k = self.K[i][j]
                kc[x, :, j % self.page], vc[x, :, j % self.page] = k, self.V[i][j]
                new = j % self.page == 0
                self.lo[x] = k if new else np.minimum(self.lo[x], k)
                self.hi[x] = k if new else np.maximum(self.hi[x], k)

    def there(self, i):
        """Whether each token's page is there."""
        x = np.array([self.table[i, j // self.page] if j // self.page < self.ldt else -1 for j in range(self.total[i])], int)
        return (x >= 0) & (x < self.pages)

    def args(self, **kw):
        p = (lambda d: None if d is None else d.ptr)
        es = self.kb.itemsize
        a = self.H.KvCache(k=self.dk_.ptr + es * self.at, v=self.dv_.ptr + es * self.at, k_ps=self.k_ps, v_ps=self.v_ps, f16=self.f16,
                           pages=self.pages, page=self.page, Hk=self.hk, dk=self.dk, dv=self.dv, lo=p(self.dlo), hi=p(self.dhi),
                           table=self.dtable.ptr, ldt=self.ldt, past=self.dpast.ptr)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    def seqs(self):
        return self.T, self.B, self.rows, self.dstart.ptr, self.dlen.ptr


def same(got, want):
    return np.array_equal(got, want, equal_nan=True)


# ------------------------------------------------------------------------------------------------ append
class Append:
    def __init__(self, H, pasts, lens, heads, hk, dk, dv, rd, pairs=0, page=32, f16=1, seed=0, pad=0, at=0, pos=None, base=1e4,
                 q=True, inplace=False, **kw):
        rng = np.random.default_rng(seed + 1)
        self.c = c = Cache(H, pasts, lens, hk, dk, dv, page, f16, seed, held=pasts, at=at, **kw)
        self.H, self.heads, self.rd, self.pairs, self.inplace = H, heads, rd, pairs, inplace
        self.freq = (base ** (-2 * np.arange(rd // 2) / max(1, rd))).astype(np.float32)
        t = c.t
        self.q = rng.standard_normal((c.rows, heads, dk)).astype(t)
        self.k, self.v = rng.standard_normal((c.rows, hk, dk)).astype(t), rng.standard_normal((c.rows, hk, dv)).astype(t)
        self.pos = None if pos is None else np.asarray(pos(c), np.int32)
        rows = lambda x: Rows(H, 1, c.rows, x[0].size, t, x[0].size + pad, 0, at, x.reshape(c.rows, -1))  # noqa: E731
        self.dq, self.dk, self.dv = rows(self.q), rows(self.k), rows(self.v)
        self.dqr = self.dq if inplace else Rows(H, 1, c.rows, heads * dk, t, heads * dk + pad, 0, at)
        self.dfreq = H.DeviceArray.from_host(self.freq if rd else np.zeros(1, np.float32))
        self.dpos = None if pos is None else H.DeviceArray.from_host(self.pos)
        self.has_q = q

    def run(self, stream=None, **kw):
        H, c = self.H, self.c
        r = H.Rotary(self.rd, self.pairs, self.dfreq.ptr, None if self.dpos is None else self.dpos.ptr)
        q, qr = (self.dq.ptr, self.dqr.ptr) if self.has_q else (None, None)
        H.check(H.lib().bnh_kv_append(c.args(**kw), r, self.dk.ptr, self.dk.ld, self.dv.ptr, self.dv.ld, q, self.dq.ld, qr,
                                      self.dqr.ld, self.heads, *c.seqs(), stream), "append")
        H.sync(stream)

    def check(self, what):
        """The rotated queries; keys, values and bounds in their places, and nothing else written. A key may differ from the
        64-bit one by its rounding, so the bounds are held to the keys that are there."""
        c = self.c
        kb, vb = c.dk_.numpy(), c.dv_.numpy()
        kc, vc = c.place(kb, c.k_ps, c.dk), c.place(vb, c.v_ps, c.dv)
        lo, hi = (c.dlo.numpy(), c.dhi.numpy()) if c.dlo else (None, None)
        if self.has_q:
            # rows that no sequence has keep what was there
            got = self.dqr.get()[0].reshape(c.rows, self.heads, c.dk)
            none = np.ones(c.rows, bool)
        for i in range(c.B):
            s, n, m = int(c.start[i]), min(c.lens[i], c.T), max(0, c.pasts[i])
            at = m + np.arange(n)
            pos = at if self.pos is None else self.pos[s:s + n]
            if self.has_q:
                want, err = R.rotate(self.q[s:s + n], pos, self.rd, self.pairs, self.freq)
                near(got[s:s + n], want, err, what + " q", c.f16)
                none[s:s + n] = False
            want, err = R.rotate(self.k[s:s + n], pos, self.rd, self.pairs, self.freq)
            for r, j in enumerate(at):
                x = c.table[i, j // c.page] if j // c.page < c.ldt else -1
                if not 0 <= x < c.pages:
                    continue
                c.K[i][j], c.V[i][j] = kc[x, :, j % c.page], vc[x, :, j % c.page]
                near(c.K[i][j], want[r], err[r], what + f" k {i} {j}", c.f16) if r in (0, n - 1) else None
                assert same(c.V[i][j], self.v[s + r]), (what, i, j)
            keep = c.there(i)[m:m + n]
            near(c.K[i][m:m + n][keep], want[keep], err[keep], what + " k", c.f16)
            c.store(i, m, m + n)
        assert same(kb, c.kb) and same(vb, c.vb), what + ": written outside"
        if lo is not None:
            assert same(lo, c.lo) and same(hi, c.hi), what + ": bounds"
        if self.has_q:
            assert same(got[none], self.q[none] if self.inplace else np.full_like(got[none], 7)), what + ": rows of nobody"


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dk,dv,rd,pairs", [(128, 128, 128, 0), (128, 64, 64, 1), (64, 128, 32, 0), (256, 256, 256, 0), (256, 8, 128, 1),
                                            (70, 97, 42, 1), (70, 97, 42, 0), (33, 31, 32, 0), (33, 31, 32, 1), (1, 1, 0, 0),
                                            (2, 3, 2, 1), (255, 255, 254, 0), (48, 40, 0, 0), (16, 16, 16, 1), (80, 80, 16, 0)])
def test_append_widths(hip, f16, dk, dv, rd, pairs):
    say(f"append {dk} {dv} rd {rd} pairs {pairs} f16 {f16}")
    a = Append(hip, [0, 40, 31, 7], [70, 1, 33, 0], 6, 2, dk, dv, rd, pairs, 32, f16, seed=dk + rd)
    a.run()
    a.check("widths")


@pytest.mark.parametrize("page", [16, 64, 128, 1024])
@pytest.mark.parametrize("heads,hk", [(1, 1), (12, 12), (20, 1), (8, 4)])
def test_append_pages_and_heads(hip, page, heads, hk):
    say(f"append page {page} heads {heads} {hk}")
    a = Append(hip, [0, page - 1, page, 5 * page + 3, 200], [page, 1, page + 1, 2 * page, 3], heads, hk, 64, 48, 64, 0, page, 1, extra=64,
               seed=page)
    a.run()
    a.check("pages")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("pad,at,extra", [(8, 8, 16), (3, 0, 0), (8, 1, 8), (0, 0, 5)])
def test_append_strides(hip, f16, pad, at, extra):
    """Rows and pages apart from each other, aligned or not; in place; keys alone; no bounds; no rotation's struct."""
    say(f"append strides {pad} {at} {extra} f16 {f16}")
    for kw in (dict(), dict(inplace=True), dict(q=False), dict(bounds=False)):
        a = Append(hip, [5, 64], [40, 9], 4, 2, 64, 32, 32, 0, 32, f16, pad=pad, at=at, extra=extra, seed=at, **kw)
        a.run()
        a.check(str(kw))


def test_append_positions(hip):
    """Positions of their own, far and negative ones: an angle is as exact there."""
    for f16 in (0, 1):
        for pairs in (0, 1):
            say(f"append positions f16 {f16} pairs {pairs}")

            def pos(c):
                p = np.random.default_rng(3).integers(-2 ** 31, 2 ** 31, c.rows)
                p[:3] = 2 ** 31 - 1, -2 ** 31, 0
                return p

            a = Append(hip, [3, 0], [50, 20], 2, 1, 64, 16, 64, pairs, 16, f16, pos=pos, base=1e3)
            a.run()
            a.check("positions")


def test_append_in_pieces(hip):
    """A sequence's rows in calls of any lengths leave what one call leaves, bounds too."""
    say("append in pieces")
    n, page = 150, 32
    one = Append(hip, [0], [n], 2, 2, 48, 40, 48, 0, page, 1, seed=5)
    one.run()
    one.check("one")
    c = Append(hip, [0], [n], 2, 2, 48, 40, 48, 0, page, 1, seed=5)
    at = 0
    for m in (1, 1, 30, 1, 31, 40, 2, 44):
        c.c.dpast.upload(np.array([at], np.int32))
        c.c.dstart.upload(np.array([at], np.int32))
        c.c.dlen.upload(np.array([m], np.int32))
        c.run()
        at += m
    assert at == n
    for x, y in ((one.c.dk_, c.c.dk_), (one.c.dv_, c.c.dv_), (one.c.dlo, c.c.dlo), (one.c.dhi, c.c.dhi)):
        assert same(x.numpy(), y.numpy())
    assert same(one.dqr.get(), c.dqr.get())


def test_append_not_there(hip):
    """Pages that are not there, tokens past the table, a past below 0, lengths past T and the buffers, starts outside."""
    say("append not there")
    a = Append(hip, [40, 0, 60], [100, 30, 8], 4, 2, 32, 32, 32, 0, 16, 1, gone=[(0, 3), (0, 8), (2, 4)], more=0)
    a.run()
    a.check("gone")
    for f16 in (0, 1):
        a = Append(hip, [5, 0, 9, 3], [20, 20, 20, 20], 2, 2, 32, 32, 32, 0, 16, f16, T=20)
        c = a.c
        c.dpast.upload(np.array([5, -7, 9, 3], np.int32))
        c.dlen.upload(np.array([500, 20, -3, 20], np.int32))
        c.start = np.array([0, 21, 42, c.rows], np.int32)
        c.dstart.upload(c.start)
        c.pasts, c.lens = [5, 0, 9, 3], [20, 20, 0, 0]
        a.run()
        a.check("cut")


def test_append_not_finite(hip):
    """A NaN among a page's keys stays in its bounds, an infinity is one of them."""
    say("append not finite")
    a = Append(hip, [0, 10], [40, 40], 2, 2, 32, 32, 0, 0, 16, 1)
    a.k[3, 0, 5], a.k[20, 1, 7], a.k[21, 1, 8] = np.nan, np.inf, -np.inf
    a.dk = Rows(hip, 1, a.c.rows, 64, np.float16, 64, 0, 0, a.k.reshape(a.c.rows, -1))
    a.run()
    a.check("not finite")


# ------------------------------------------------------------------------------------------------ attention
class Attn:
    def __init__(self, H, pasts, lens, heads, hk, dk, dv, page=32, f16=1, seed=0, window=0, pad=0, qstd=1.0, scale=None, sel=None,
                 at=0, **kw):
        rng = np.random.default_rng(seed + 2)
        self.c = c = Cache(H, pasts, lens, hk, dk, dv, page, f16, seed, at=at, **kw)
        self.H, self.heads, self.window = H, heads, window
        self.scale = dk ** -0.5 if scale is None else scale
        self.q = (rng.standard_normal((c.rows, heads, dk)) * qstd).astype(c.t)
        self.dq = Rows(H, 1, c.rows, heads * dk, c.t, heads * dk + pad, 0, at, self.q.reshape(c.rows, -1))
        self.do = Rows(H, 1, c.rows, heads * dv, c.t, heads * dv + pad, 0, at)
        self.sel = None if sel is None else np.asarray(sel(c), np.int32)
        self.dsel = None if sel is None else H.DeviceArray.from_host(self.sel)

    def args(self):
        return self.H.KvAttn(q=self.dq.ptr, ldq=self.dq.ld, o=self.do.ptr, ldo=self.do.ld, H=self.heads, scale=self.scale,
                             window=self.window, sel=None if self.sel is None else self.dsel.ptr,
                             nsel=0 if self.sel is None else self.sel.shape[-1])

    def run(self, stream=None):
        H, c, L, a = self.H, self.c, self.H.lib(), self.args()
        wb = L.bnh_kv_attn_work_bytes(c.args(), a, *c.seqs()[:3])
        ws = H.DeviceArray.from_host(np.full(wb + 256, 0xff, np.uint8))
        H.check(L.bnh_kv_attn(c.args(), a, *c.seqs(), ws.ptr if wb else None, wb, stream), "attn")
        H.sync(stream)
        assert (ws.numpy()[wb:] == 0xff).all(), "written past the workspace"

    def seen(self, i, n):
        """[n][Hk][tokens] of sequence i"""
        c = self.c
        j, at = np.arange(c.total[i]), max(0, c.pasts[i]) + np.arange(n)
        seen = c.there(i)[None] & (j <= at[:, None]) & (j > at[:, None] - (self.window or 1 << 40))
        seen = np.repeat(seen[:, None], c.hk, 1)
        if self.sel is not None:
            for r in range(n):
                for g in range(c.hk):
                    s = self.sel[c.start[i] + r, g].astype(int)
                    up = np.concatenate([[-1], s[:-1]])
                    keep = s[(s > up) & (s >= 0)]
                    seen[r, g] &= np.isin(j // c.page, keep)
        return seen

    def check(self, what, part=None):
        c = self.c
        got = self.do.get()[0].reshape(c.rows, self.heads, c.dv)
        none = np.ones(c.rows, bool)
        part = (ONE if c.f16 else 0) if part is None else part
        for i in range(c.B):
            s, n = int(c.start[i]), min(c.lens[i], c.T)
            if n < 1:
                continue
            o, err = R.attention(self.q[s:s + n], c.K[i], c.V[i], self.seen(i, n), self.scale, part)
            near(got[s:s + n], o, err, what + f" {i}", c.f16)
            none[s:s + n] = False
        assert (got[none] == 7).all(), what + ": rows of nobody"


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (32, 32), (256, 256), (64, 97), (70, 128), (1, 1), (33, 200), (250, 24), (96, 96),
                                   (16, 128), (128, 16), (120, 72)])
def test_attn_widths(hip, f16, dk, dv):
    say(f"attn {dk} {dv} f16 {f16}")
    a = Attn(hip, [0, 75, 200, 31], [40, 1, 90, 0], 4, 2, dk, dv, 32, f16, seed=dk + dv)
    a.run()
    a.check("widths")
    a = Attn(hip, [0, 31, 32, 500], [1, 1, 1, 1], 4, 4, dk, dv, 16, f16, seed=dk)
    a.run()
    a.check("one row", TWO if f16 else 0)


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("heads,hk", [(1, 1), (12, 12), (12, 4), (20, 1), (33, 1), (8, 2)])
@pytest.mark.parametrize("n", [1, 3, 17, 100])
def test_attn_heads(hip, f16, heads, hk, n):
    say(f"attn heads {heads} {hk} rows {n} f16 {f16}")
    a = Attn(hip, [0, 150, 33], [n, n, max(1, n // 2)], heads, hk, 64, 64, 64, f16, seed=heads + n)
    a.run()
    a.check("heads")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("window", [0, 1, 16, 40, 200, 100000])
def test_attn_windows_and_pages(hip, f16, page, window):
    say(f"attn page {page} window {window} f16 {f16}")
    a = Attn(hip, [0, 130, 600], [130, 70, 1], 4, 2, 64, 64, page, f16, window=window, extra=32, seed=window)
    a.run()
    a.check("windows")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("pad,at,extra", [(8, 8, 16), (3, 0, 0), (8, 1, 8), (0, 0, 5)])
def test_attn_strides(hip, f16, pad, at, extra):
    say(f"attn strides {pad} {at} {extra} f16 {f16}")
    for n in (1, 50):
        a = Attn(hip, [100, 0], [n, n], 4, 2, 64, 128, 32, f16, pad=pad, at=at, extra=extra, seed=at)
        a.run()
        a.check("strides")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_attn_long(hip, f16, n):
    """Tokens enough for many parts, of sequences much shorter than the table is wide too."""
    say(f"attn long rows {n} f16 {f16}")
    a = Attn(hip, [5000, 3, 1200], [n, n, 1], 4, 2, 128, 128, 64, f16, seed=n, more=30)
    a.run()
    a.check("long")


@pytest.mark.parametrize("f16", [0, 1])
def test_attn_not_there(hip, f16):
    """Pages that are not there in the middle and at the ends, all of a row's, tokens past the table; lengths, pasts and starts
    outside."""
    say(f"attn not there f16 {f16}")
    for n in (1, 40):
        a = Attn(hip, [100, 100, 40, 0], [n, n, n, n], 4, 2, 64, 64, 16, f16, gone=[(0, 0), (0, 3), (0, 4), (1, 6), (1, 7), (1, 8)] +
                 [(2, x) for x in range(2 + -(-n // 16))], more=0)
        a.run()
        a.check("gone")
    a = Attn(hip, [64, 0], [70, 70], 2, 2, 64, 64, 16, f16, window=20, gone=[(0, x) for x in range(4, 7)])
    a.run()
    a.check("rows of nothing")
    a = Attn(hip, [30, 30], [50, 50], 2, 1, 64, 64, 16, f16)
    a.c.ldt = 4  # of a wider table: the second sequence's row of it begins within the first's
    a.c.table = a.c.table.ravel()[:8].reshape(2, 4)
    a.run()
    a.c.total = [80, 80]
    a.c.K[1], a.c.V[1] = a.c.K[0].copy(), a.c.V[0].copy()
    for j in range(80):
        x = a.c.table[1, j // 16] if j < 64 else -1
        if 0 <= x < a.c.pages:
            a.c.K[1][j], a.c.V[1][j] = (a.c.place(b, p, 64)[x, :, j % 16] for b, p in ((a.c.kb, a.c.k_ps), (a.c.vb, a.c.v_ps)))
    a.check("past the table")
    a = Attn(hip, [20, 0, 9, 3], [20, 20, 20, 20], 2, 2, 32, 32, 16, f16, T=20)
    c = a.c
    c.dpast.upload(np.array([20, -7, 9, 3], np.int32))
    c.dlen.upload(np.array([500, 20, -3, 20], np.int32))
    c.start = np.array([0, 21, 42, c.rows], np.int32)
    c.dstart.upload(c.start)
    c.lens = [20, 20, 0, 0]
    a.run()
    a.check("cut")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dv", [64, 97])
def test_attn_not_finite(hip, f16, dv):
    """Infinities and NaNs of later tokens, of a window's earlier ones and of other heads reach no row that does not see them."""
    for bad in (np.nan, np.inf):
        for where in ("K", "V"):
            for window in (0, 25):
                def edit(c):
                    for i, j in ((0, 60), (0, 61), (1, 150)):
                        getattr(c, where)[i][j, 0, 3] = bad

                say(f"attn not finite {bad} {where} window {window} f16 {f16}")
                a = Attn(hip, [0, 120], [130, 60], 6, 2, 64, dv, 16, f16, window=window, edit=edit, seed=dv)
                a.run()
                c = a.c
                got = a.do.get()[0].astype(np.float64).reshape(c.rows, 6, dv)
                for i in range(2):
                    s, n = int(c.start[i]), c.lens[i]
                    seen = a.seen(i, n)
                    x = c.K[i] if where == "K" else c.V[i]
                    hit = (seen & ~np.isfinite(x).all(-1).T).any(-1)  # [n][Hk]
                    with np.errstate(all="ignore"):
                        o, err = R.attention(a.q[s:s + n], np.nan_to_num(c.K[i], posinf=0), c.V[i], seen, a.scale, ONE if f16 else 0)
                    hit = np.repeat(hit, 3, 1)
                    near(got[s:s + n][~hit], o[~hit], err[~hit], "unhit", f16)
                    if where == "V":  # the column alone
                        fine = np.isfinite(o)
                        near(got[s:s + n][fine], o[fine], err[fine], "other columns", f16)
                        assert not np.isfinite(got[s:s + n][~fine]).any()
                        if bad == np.inf:
                            assert (got[s:s + n][~fine] == np.inf).all()
                    elif bad != bad:
                        assert np.isnan(got[s:s + n][hit]).all()


@pytest.mark.parametrize("f16", [0, 1])
def test_attn_extreme_scores(hip, f16):
    """Large and equal scores, all of the weight on one token, scores of -inf, a negative and a zero scale."""
    say(f"attn extreme f16 {f16}")
    for n in (1, 70):
        for kw in (dict(qstd=30.0, std=30.0), dict(scale=0.0), dict(scale=-0.3), dict(qstd=0.0), dict(scale=20.0)):
            a = Attn(hip, [90, 0], [n, n], 4, 2, 64, 64, 32, f16, seed=n, **kw)
            a.run()
            a.check(str(kw))

    def edit(c):  # keys whose product with any positive query is -inf: as if they were not there
        c.K[0][:40, 0, 0] = -np.inf
        c.K[1][:, :, 0] = -np.inf

    a = Attn(hip, [60, 20], [30, 5], 4, 2, 64, 64, 16, f16, edit=edit)
    a.q = np.abs(a.q)
    a.dq = Rows(hip, 1, a.c.rows, 256, a.c.t, 256, 0, 0, a.q.reshape(a.c.rows, -1))
    a.run()
    got = a.do.get()[0].reshape(a.c.rows, 4, 64)
    assert (got[a.c.start[1]:a.c.start[1] + 5] == 0).all()
    seen = a.seen(0, 30)
    seen[:, 0, :40] = False
    o, err = R.attention(a.q[:30], a.c.K[0], a.c.V[0], seen, a.scale, ONE if f16 else 0)
    near(got[:30], o, err, "-inf", f16)


def test_attn_far_pages(hip):
    """Pages past 2^32 bytes and 2^31 elements into their pool."""
    H = hip
    say("attn far pages")
    hk, d, page, ps = 2, 64, 32, 1 << 28
    for n in (1, 40):
        a = Attn(hip, [80], [n], 4, hk, d, d, page, 1, seed=n)
        c = a.c
        big = [H.DeviceArray((ps * 9 + hk * page * d,), np.float16) for _ in range(2)]
        table = np.full(c.ldt, -1, np.int32)
        places = [9, 0, 8, 5, 7][:-(-c.total[0] // page)]
        table[:len(places)] = places
        for x, p in zip(c.table[0], places):
            for buf, host in zip(big, (c.kb, c.vb)):
                one = np.ascontiguousarray(host.reshape(c.pages, -1)[x])
                H.check(H.lib().bnh_memcpy_h2d(buf.ptr + 2 * p * ps, one.ctypes.data, one.nbytes))
        dt = H.DeviceArray.from_host(table)
        cache = c.args(k=big[0].ptr, v=big[1].ptr, k_ps=ps, v_ps=ps, pages=10, table=dt.ptr)
        wb = H.lib().bnh_kv_attn_work_bytes(cache, a.args(), *c.seqs()[:3])
        ws = H.DeviceArray((max(16, wb),), np.uint8)
        H.check(H.lib().bnh_kv_attn(cache, a.args(), *c.seqs(), ws.ptr, wb, None))
        H.sync()
        a.check("far")
        # the same through append: a row more into the last page
        if n == 1:
            r = H.DeviceArray.from_host(np.arange(2 * hk * d, dtype=np.float16))
            past = H.DeviceArray.from_host(np.array([81], np.int32))
            one = H.DeviceArray.from_host(np.array([1], np.int32))
            cache.past, cache.lo, cache.hi = past.ptr, None, None
            H.check(H.lib().bnh_kv_append(cache, None, r.ptr, hk * d, r.ptr + 2 * hk * d, hk * d, None, 0, None, 0, 0, 1, 1, 1, None,
                                          one.ptr, None))
            H.sync()
            got = np.empty(d, np.float16)
            at = 8 * ps + (page + 81 % page) * d
            for buf, first in zip(big, (d, (hk + 1) * d)):
                H.check(H.lib().bnh_memcpy_d2h(got.ctypes.data, buf.ptr + 2 * at, 2 * d))
                assert np.array_equal(got, np.arange(first, first + d))


# ------------------------------------------------------------------------------------------------ selection
def pick(a, first, last, n, stream=None):
    """bnh_kv_select of an Attn's rows -> [rows][Hk][n]"""
    H, c, L = a.H, a.c, a.H.lib()
    sel = H.DeviceArray.from_host(np.full((c.rows, c.hk, n), -7, np.int32))
    p = a.args()
    p.sel, p.nsel = sel.ptr, n
    wb = L.bnh_kv_select_work_bytes(c.args(), p, *c.seqs()[:3])
    ws = H.DeviceArray.from_host(np.full(wb + 256, 0xff, np.uint8))
    H.check(L.bnh_kv_select(c.args(), p, first, last, *c.seqs(), ws.ptr, wb, stream), "select")
    H.sync(stream)
    assert (ws.numpy()[wb:] == 0xff).all(), "written past the workspace"
    return sel.numpy()


def check_pick(a, got, first, last, n, what):
    c = a.c
    lo, hi = c.dlo.numpy(), c.dhi.numpy()
    none = np.ones(c.rows, bool)
    for i in range(c.B):
        there = (c.table[i] >= 0) & (c.table[i] < c.pages)
        x = np.where(there, c.table[i], 0)
        for r in range(min(c.lens[i], c.T)):
            row = int(c.start[i]) + r
            want = R.select(a.q[row], lo[x], hi[x], there, max(0, c.pasts[i]) + r, c.page, a.window, first, last, n)
            assert np.array_equal(got[row], want), (what, i, r)
            none[row] = False
    assert (got[none] == -7).all(), what + ": rows of nobody"


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dk", [128, 64, 70, 1, 256, 200])
@pytest.mark.parametrize("heads,hk", [(2, 2), (6, 2), (40, 1)])
def test_select(hip, f16, dk, heads, hk):
    say(f"select dk {dk} heads {heads} {hk} f16 {f16}")
    a = Attn(hip, [0, 700, 333], [50, 1, 20], heads, hk, dk, 16, 16, f16, seed=dk + heads, gone=[(1, 3), (1, 30), (2, 0)])
    for first, last, n in ((1, 2, 8), (0, 0, 1), (0, 1, 5), (3, 3, 6), (2, 5, 200)):
        check_pick(a, pick(a, first, last, n), first, last, n, f"{first} {last} {n}")


def test_select_many_pages(hip):
    """More pages than a block has threads, and than one pass takes; a window that leaves some; ties."""
    for window in (0, 9000, 100):
        say(f"select many window {window}")
        a = Attn(hip, [20000, 5000], [2, 3], 2, 1, 24, 8, 16, 1, window=window, seed=9)
        for n in (4, 64, 700):
            check_pick(a, pick(a, 1, 2, n), 1, 2, n, f"many {n}")

    def edit(c):  # keys of a few values: most bounds and scores are equal
        c.K[0][:] = np.round(c.K[0] * 0.6)

    a = Attn(hip, [6000], [2], 2, 1, 2, 8, 16, 1, edit=edit)
    a.q[:] = np.sign(a.q)
    a.dq = Rows(hip, 1, a.c.rows, 4, np.float16, 4, 0, 0, a.q.reshape(a.c.rows, -1))
    for n in (3, 50, 300):
        check_pick(a, pick(a, 1, 1, n), 1, 1, n, f"ties {n}")
    a.q[:] = 0
    a.dq = Rows(hip, 1, a.c.rows, 4, np.float16, 4, 0, 0, a.q.reshape(a.c.rows, -1))
    check_pick(a, pick(a, 1, 1, 20), 1, 1, 20, "all equal")


@pytest.mark.parametrize("f16", [0, 1])
def test_select_not_finite(hip, f16):
    """Bounds that are not finite: NaN sums are the lowest, infinities rank as they are."""
    say(f"select not finite f16 {f16}")

    def edit(c):
        c.K[0][100, 0, 3], c.K[0][200, 0, 4], c.K[0][300, 0, 4], c.K[0][301, 0, 4] = np.nan, np.inf, -np.inf, np.inf

    a = Attn(hip, [700], [4], 4, 2, 32, 16, 16, f16, edit=edit, seed=2)
    a.q[1, 1, 5], a.q[2, 0, 4] = np.nan, 0
    a.dq = Rows(hip, 1, a.c.rows, 128, a.c.t, 128, 0, 0, a.q.reshape(a.c.rows, -1))
    for n in (3, 20, 43, 60):
        check_pick(a, pick(a, 1, 1, n), 1, 1, n, f"not finite {n}")


def test_select_is_a_bound(hip):
    """No token's product with the queries is above its page's score."""
    say("select bound")
    a = Attn(hip, [300], [1], 6, 2, 48, 16, 32, 0, seed=4)
    c = a.c
    x = c.table[0][:10]
    s = R.scores(a.q[0], c.dlo.numpy()[x], c.dhi.numpy()[x])
    q = a.q[0].astype(np.float64).reshape(2, 3, 48).sum(1)
    for j in range(301):
        assert ((c.K[0][j].astype(np.float64) * q).sum(-1) <= s[:, j // 32] + 1e-12).all()


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("heads,hk", [(2, 2), (12, 4), (40, 1)])
def test_attn_selected(hip, f16, page, heads, hk):
    """Selections with -1, entries outside the table, out of order, twice, and of pages that the row does not see or that are
    not there."""
    def sel(c):
        s = np.sort(np.random.default_rng(page).integers(-2, c.ldt + 2, (c.rows, hk, 9)), -1)  # some twice
        s[::3, :, 5:] = -1
        s[1::5, 0, 2] = 1
        s[::7] = -1
        return s

    say(f"attn selected page {page} heads {heads} {hk} f16 {f16}")
    a = Attn(hip, [8 * page + 5, 0, 11 * page], [1, 70, 20], heads, hk, 64, 80, page, f16, sel=sel, gone=[(2, 4)], seed=page)
    a.run()
    a.check("selected", TWO if f16 else 0)


def test_attn_selected_all(hip):
    """All pages selected is attention without a selection: within both bounds; many of them are cut into parts."""
    for f16 in (0, 1):
        say(f"selected all f16 {f16}")
        a = Attn(hip, [3100, 900], [2, 1], 4, 2, 128, 128, 32, f16, sel=lambda c: np.tile(np.arange(c.ldt), (c.rows, 2, 1)))
        a.run()
        a.check("all", TWO if f16 else 0)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("f16", [0, 1])
def test_together(hip, f16):
    """Rows into the cache, their selection and attention over it, call by call as a program makes them: an archive and then
    live rows, dense and selected."""
    H, L = hip, hip.lib()
    hk, heads, d, page, n = 2, 6, 64, 16, 6
    lens = [[70, 33, 1], [1, 1, 1], [5, 0, 9], [1, 1, 1]]
    total = np.sum(lens, 0)
    rng = np.random.default_rng(6)
    t = typ(f16)
    c = Cache(H, [0, 0, 0], list(total), hk, d, d, page, f16, held=[0, 0, 0])
    freq = (100.0 ** (-2 * np.arange(d // 2) / d)).astype(np.float32)
    dfreq = H.DeviceArray.from_host(freq)
    rot = H.Rotary(d, 0, dfreq.ptr, None)
    past = np.zeros(3, int)
    keys, vals = ([np.zeros((0, hk, d), t) for _ in range(3)] for _ in range(2))
    for step, new in enumerate(lens):
        say(f"together step {step} f16 {f16}")
        rows, T = sum(new), max(new)
        x = rng.standard_normal((rows, (heads + 2 * hk) * d)).astype(t)
        dx, start = H.DeviceArray.from_host(x), np.cumsum([0] + new[:-1])
        dqr, do = H.DeviceArray((rows, heads * d), t), H.DeviceArray((rows, heads * d), t)
        dsel = H.DeviceArray((rows, hk, n), np.int32)
        ds, dl, dp = (H.DeviceArray.from_host(np.asarray(y, np.int32)) for y in (start, new, past))
        cache = c.args(past=dp.ptr)
        es, ld = x.itemsize, x.shape[1]
        seqs = (T, 3, rows, ds.ptr, dl.ptr)
        H.check(L.bnh_kv_append(cache, rot, dx.ptr + es * heads * d, ld, dx.ptr + es * (heads + hk) * d, ld, dx.ptr, ld, dqr.ptr,
                                heads * d, heads, *seqs, None))
        a = H.KvAttn(q=dqr.ptr, ldq=heads * d, o=do.ptr, ldo=heads * d, H=heads, scale=d ** -0.5, window=0)
        b = H.KvAttn(q=dqr.ptr, ldq=heads * d, o=do.ptr, ldo=heads * d, H=heads, scale=d ** -0.5, window=0, sel=dsel.ptr, nsel=n)
        wb = max(L.bnh_kv_attn_work_bytes(cache, a, *seqs[:3]), L.bnh_kv_attn_work_bytes(cache, b, *seqs[:3]),
                 L.bnh_kv_select_work_bytes(cache, b, *seqs[:3]))
        ws = H.DeviceArray((wb,), np.uint8)
        H.check(L.bnh_kv_attn(cache, a, *seqs, ws.ptr, wb, None))
        H.sync()
        dense = do.numpy().reshape(rows, heads, d)
        H.check(L.bnh_kv_select(cache, b, 1, 2, *seqs, ws.ptr, wb, None))
        H.check(L.bnh_kv_attn(cache, b, *seqs, ws.ptr, wb, None))
        H.sync()
        kc = c.place(c.dk_.numpy(), c.k_ps, d)
        few, sel, qr = do.numpy().reshape(rows, heads, d), dsel.numpy(), dqr.numpy().reshape(rows, heads, d)
        for i in range(3):
            r = slice(start[i], start[i] + new[i])
            at = past[i] + np.arange(new[i])
            zk, zv = x[r, heads * d:(heads + hk) * d].reshape(-1, hk, d), x[r, (heads + hk) * d:].reshape(-1, hk, d)
            stored = np.array([kc[c.table[i, y // page], :, y % page] for y in at], t).reshape(-1, hk, d)
            want, err = R.rotate(zk, at, d, 0, freq)
            near(stored, want, err, "k", f16)
            keys[i], vals[i] = np.concatenate([keys[i], stored]), np.concatenate([vals[i], zv])
            want, err = R.rotate(x[r, :heads * d].reshape(-1, heads, d), at, d, 0, freq)
            near(qr[r], want, err, "q", f16)
            if not new[i]:
                continue
            j = np.arange(len(keys[i]))
            seen = np.repeat((j <= at[:, None])[:, None], hk, 1)
            for got, s in ((dense, seen), (few, seen & np.stack([np.isin(j // page, sel[row][g]) for row in range(r.start, r.stop)
                                                                 for g in range(hk)]).reshape(-1, hk, len(j)))):
                o, e = R.attention(qr[r], keys[i], vals[i], s, d ** -0.5, ONE if f16 else 0)
                near(got[r], o, e, "o", f16)
            lo, hi = c.dlo.numpy(), c.dhi.numpy()
            there = c.table[i] >= 0
            xs = np.where((c.table[i] >= 0) & (c.table[i] < c.pages), c.table[i], 0)
            there &= c.table[i] < c.pages
            for k, row in enumerate(range(r.start, r.stop)):
                assert np.array_equal(sel[row], R.select(qr[row], lo[xs], hi[xs], there, at[k], page, 0, 1, 2, n))
        past = past + new
