"""The selection of pages where scores are not finite, and where its launches are cut."""
import numpy as np
import pytest

import cache_ref as R
from test_gpu_cache import TWO, Attn, Rows, check_pick, pick
from test_gpu_context import near, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("tokens", [300, 700, 3000, 70000])
def test_forced_before_infinite(hip, f16, tokens):
    """The first pages and the row's own are taken always, also where more pages than there is room for have bounds of +infinity:
    few pages, a pass of them, and more than one pass."""
    say(f"forced tokens {tokens} f16 {f16}")

    def edit(c):  # an infinite key in every third page
        c.K[0][5::48, :, 4] = np.inf

    a = Attn(hip, [tokens - 4], [4], 4, 2, 24, 8, 16, f16, edit=edit, seed=tokens)
    a.q[..., 4] = np.abs(a.q[..., 4]) + 1
    a.dq = Rows(hip, 1, a.c.rows, 96, a.c.t, 96, 0, 0, a.q.reshape(a.c.rows, -1))
    own = (tokens - 4 + np.arange(4)) // 16
    some = (tokens + 15) // 16 // 3
    for first, last, n in ((1, 2, 3), (1, 2, 4), (0, 1, 1), (0, 1, 2), (2, 1, 9), (0, 0, 5), (1, 1, some - 1), (1, 1, some + 7)):
        got = pick(a, first, last, n)
        for r in range(4):
            for g in range(2):
                s = got[r, g][got[r, g] >= 0]
                assert (np.diff(s) > 0).all()
                assert set(range(first)) | {own[r] - x for x in range(last)} <= set(s.tolist()), (first, last, n, r, g)
        check_pick(a, got, first, last, n, f"forced {first} {last} {n}")


@pytest.mark.parametrize("f16", [0, 1])
def test_an_infinite_key_that_the_row_does_not_see(hip, f16):
    """A window that begins within a page: an infinite key ahead of it makes the page's bound infinite, and does not cost the row its
    own page."""
    say(f"infinite key ahead of the window f16 {f16}")

    def edit(c):
        c.K[0][640:644, :, 4] = np.inf

    a = Attn(hip, [999], [1], 2, 2, 32, 32, 16, f16, window=350, edit=edit, seed=3)  # tokens from 650 on: page 40's last six
    a.q[..., 4] = np.abs(a.q[..., 4]) + 1
    a.dq = Rows(hip, 1, a.c.rows, 64, a.c.t, 64, 0, 0, a.q.reshape(a.c.rows, -1))
    sel = pick(a, 0, 1, 1)
    assert (sel[0] == 62).all()
    sel = pick(a, 0, 1, 2)
    assert (sel[0] == [40, 62]).all()
    b = Attn(hip, [999], [1], 2, 2, 32, 32, 16, f16, window=350, edit=edit, seed=3, sel=lambda c: sel)
    b.q[:], b.dq = a.q, a.dq
    b.run()
    got = b.do.get()[0][:1].reshape(1, 2, 32)
    o, err = R.attention(b.q[:1], np.nan_to_num(b.c.K[0], posinf=0), b.c.V[0], b.seen(0, 1), b.scale, TWO if f16 else 0)
    assert np.isfinite(got).all()
    near(got, o, err, "selected", f16)


def test_more_rows_than_a_launch_has_threads_for(hip):
    """Rows and heads whose choices, a block of 512 threads each, would be 2^32 threads and more in one launch."""
    say("rows past a launch")
    L, hk, rows = hip.lib(), 4, (1 << 21) + 3
    z = hip.DeviceArray.zeros
    q, sel, kv = z((rows, hk), np.float16), hip.DeviceArray((rows, hk, 2), np.int32), z((hk * 16,), np.float16)
    sel.fill(0x7f)
    table, past = z((1,), np.int32), z((1,), np.int32)
    c = hip.KvCache(k=kv.ptr, v=kv.ptr, k_ps=hk * 16, v_ps=hk * 16, f16=1, pages=1, page=16, Hk=hk, dk=1, dv=1, lo=kv.ptr, hi=kv.ptr,
                    table=table.ptr, ldt=1, past=past.ptr)
    a = hip.KvAttn(q=q.ptr, ldq=hk, H=hk, scale=1, sel=sel.ptr, nsel=2)
    wb = L.bnh_kv_select_work_bytes(c, a, rows, 1, rows)
    ws = hip.DeviceArray((wb,), np.uint8)
    hip.check(L.bnh_kv_select(c, a, 0, 1, rows, 1, rows, None, None, ws.ptr, wb, None))
    hip.sync()
    got = sel.numpy()
    assert (got[..., 0] == 0).all() and (got[..., 1] == -1).all()


def test_launches_that_begin_within_a_sequence(hip):
    """A table wide enough for a few rows' scores to fill the workspace: launches begin in the middle of sequences, and use it
    again."""
    say("launches within a sequence")
    a = Attn(hip, [200, 0, 33, 5], [23, 20, 0, 17], 12, 12, 8, 8, 16, 1, seed=1, more=70000)
    c, L = a.c, hip.lib()
    p = a.args()
    p.nsel = 6
    wb = L.bnh_kv_select_work_bytes(c.args(), p, *c.seqs()[:3])
    per = wb // (8 * c.hk * c.ldt)
    assert 1 < per < 20 and c.T % per
    got = pick(a, 1, 2, 6)  # the workspace's end and rows of nobody are looked at by what follows and by pick
    lo, hi = c.dlo.numpy(), c.dhi.numpy()
    none = np.ones(c.rows, bool)
    for i in range(c.B):
        m = -(-c.total[i] // 16)
        x = c.table[i, :m]
        for r in range(c.lens[i]):
            row = int(c.start[i]) + r
            want = R.select(a.q[row], lo[x], hi[x], np.ones(m, bool), c.pasts[i] + r, 16, 0, 1, 2, 6)
            assert np.array_equal(got[row], want), (i, r)
            none[row] = False
    assert (got[none] == -7).all()
