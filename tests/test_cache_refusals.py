"""What the cached-attention operators refuse, on the host, before anything is launched (the pointers are never read)."""
import pytest

from bnneon import hip as H
from test_context_refusals import P, refused


def cache(**kw):
    a = H.KvCache(k=P, v=P, k_ps=2 * 32 * 24, v_ps=2 * 32 * 40, f16=1, pages=9, page=32, Hk=2, dk=24, dv=40, lo=P, hi=P, table=P,
                  ldt=7, past=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attn(**kw):
    a = H.KvAttn(q=P, ldq=96, o=P, ldo=160, H=4, scale=0.2, window=0, sel=None, nsel=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_CACHE = [dict(k=None), dict(v=None), dict(table=None), dict(past=None), dict(k_ps=2 * 32 * 24 - 1), dict(v_ps=2 * 32 * 40 - 1),
             dict(f16=2), dict(pages=0), dict(page=8), dict(page=48), dict(page=2048), dict(Hk=0), dict(dk=0), dict(dk=257),
             dict(dv=0), dict(dv=257), dict(lo=None), dict(hi=None), dict(ldt=0), dict(ldt=1 << 26), dict(k=P + 1),
             dict(v=P + 1), dict(lo=P + 1), dict(table=P + 2), dict(past=P + 2), dict(f16=0, k=P + 2)]


def append(c=None, r=(24, 0, P, P), k=P, ldk=48, v=P, ldv=80, q=P, ldq=96, qr=P + (1 << 16), ldr=96, heads=4, T=5, B=2, rows=10,
           start=P, n=P):
    return H.lib().bnh_kv_append(cache() if c is None else c, H.Rotary(*r) if r else None, k, ldk, v, ldv, q, ldq, qr, ldr, heads,
                                 T, B, rows, start, n, None)


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_cache_refused(kw):
    refused(append(cache(**kw)))
    refused(H.lib().bnh_kv_attn(cache(**kw), attn(), 5, 2, 10, P, P, P, 1 << 40, None))
    refused(H.lib().bnh_kv_select(cache(**kw), attn(sel=P, nsel=4), 1, 1, 5, 2, 10, P, P, P, 1 << 40, None))


@pytest.mark.parametrize("kw", [
    dict(r=(25, 0, P, P)), dict(r=(26, 0, P, P)), dict(r=(-2, 0, P, P)), dict(r=(24, 2, P, P)), dict(r=(24, 0, None, P)),
    dict(r=(24, 0, P + 2, P)), dict(r=(24, 0, P, P + 1)), dict(k=None), dict(v=None), dict(ldk=47), dict(ldv=79), dict(ldq=95),
    dict(ldr=95), dict(q=None), dict(qr=None), dict(heads=0), dict(heads=3), dict(qr=P, ldr=104), dict(k=P + 1), dict(v=P + 1),
    dict(q=P + 1), dict(qr=P + 1), dict(T=0), dict(T=(1 << 30) + 1), dict(B=0), dict(B=1 << 23), dict(rows=0),
    dict(start=None, rows=9), dict(start=P + 2), dict(n=P + 2)], ids=str)
def test_append_refused(kw):
    refused(append(**kw))
    refused(H.lib().bnh_kv_append(None, None, P, 48, P, 80, None, 0, None, 0, 4, 5, 2, 10, P, P, None))


BAD_ATTN = [dict(q=None), dict(ldq=95), dict(H=0), dict(H=3), dict(H=1 << 17), dict(window=-1), dict(q=P + 1)]


@pytest.mark.parametrize("kw", BAD_ATTN + [dict(o=None), dict(ldo=159), dict(o=P + 1), dict(nsel=-1), dict(nsel=4),
                                           dict(sel=P), dict(sel=P + 2, nsel=4), dict(sel=P, nsel=(1 << 20) + 1)], ids=str)
def test_attn_refused(kw):
    refused(H.lib().bnh_kv_attn(cache(), attn(**kw), 5, 2, 10, P, P, P, 1 << 40, None))


@pytest.mark.parametrize("kw", BAD_ATTN + [dict(sel=None), dict(nsel=0), dict(sel=P + 2), dict(nsel=(1 << 20) + 1)], ids=str)
def test_select_refused(kw):
    refused(H.lib().bnh_kv_select(cache(), attn(**{**dict(sel=P, nsel=4), **kw}), 1, 1, 5, 2, 10, P, P, P, 1 << 40, None))


@pytest.mark.parametrize("first,last", [(-1, 1), (1, -1), (3, 2), (5, 0), (1 << 30, 1 << 30)])
def test_select_forced_refused(first, last):
    refused(H.lib().bnh_kv_select(cache(), attn(sel=P, nsel=4), first, last, 5, 2, 10, P, P, P, 1 << 40, None))


@pytest.mark.parametrize("T,B,rows,start", [(0, 2, 10, P), (5, 0, 10, P), (5, 2, 0, P), (5, 2, 9, None), (1, 1 << 23, 1 << 24, P),
                                            ((1 << 30) + 1, 1, 10, P)])
def test_sizes_refused(T, B, rows, start):
    refused(H.lib().bnh_kv_attn(cache(), attn(), T, B, rows, start, P, P, 1 << 60, None))
    refused(H.lib().bnh_kv_select(cache(), attn(sel=P, nsel=4), 1, 1, T, B, rows, start, P, P, 1 << 60, None))
    if rows != 9:  # the workspace does not go by where rows begin
        assert H.lib().bnh_kv_attn_work_bytes(cache(), attn(), T, B, rows) == 0
        assert b"check failed" in H.lib().bnh_last_error()
        assert H.lib().bnh_kv_select_work_bytes(cache(), attn(nsel=4), T, B, rows) == 0
        assert b"check failed" in H.lib().bnh_last_error()


def test_workspaces():
    """A call without all of its workspace is refused; few tokens need none."""
    L = H.lib()
    c, a = cache(ldt=600), attn()
    need = L.bnh_kv_attn_work_bytes(c, a, 1, 2, 2)
    assert need >= 2 * 4 * 2 * 40 * 4  # two parts at least of every head's sums
    for work, size in ((P, need - 1), (None, need), (P + 8, need)):
        refused(L.bnh_kv_attn(c, a, 1, 2, 2, P, P, work, size, None), "bnh_kv_attn")
    assert L.bnh_kv_attn_work_bytes(cache(), a, 1, 2, 2) == 0
    s = attn(sel=P, nsel=4)
    need = L.bnh_kv_select_work_bytes(c, s, 1, 2, 2)
    assert need >= 2 * 2 * 600 * 8
    for work, size in ((P, need - 1), (None, need), (P + 8, need)):
        refused(L.bnh_kv_select(c, s, 1, 1, 1, 2, 2, P, P, work, size, None), "bnh_kv_select")
    # the scores' workspace does not grow with a long call's rows
    assert L.bnh_kv_select_work_bytes(c, s, 1 << 20, 2, 1 << 21) <= 64 << 20
