"""What the temporal context operators refuse, on the host, before anything is launched (the pointers are never read)."""
import ctypes

import pytest

from bnneon import hip as H

P = 1 << 20  # an address of every alignment that is asked for


def refused(rc, *words):
    assert rc != 0
    msg = H.lib().bnh_last_error().decode()
    assert all(w in msg for w in words + ("check failed",)), msg


def norm_args(**kw):
    a = H.BlockNorm(f=P, f_ws=640, ldf=64, f16=1, post=H.Norm(1, 1e-5, P, None), gate=P, g_ws=640, ldg=64, gate_act=1,
                    scale=P, rs=1.0, x=P, x_ws=640, ldx=64, x16=0, y=P, y_ws=640, ldy=64, pre=H.Norm(1, 1e-5, P, P), n=P,
                    n_ws=640, ldn=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(f=None), dict(f=None, gate=None, scale=None, x=None), dict(y=None, n=None), dict(ldf=63), dict(ldx=63),
    dict(ldg=63), dict(ldy=63), dict(ldn=63), dict(y_ws=639), dict(n_ws=600), dict(f16=2), dict(f16=0, x16=1),
    dict(x16=2), dict(gate_act=4), dict(gate_act=-1), dict(post=H.Norm(3, 1e-5, None, None)),
    dict(pre=H.Norm(-1, 1e-5, None, None)), dict(f=P + 1), dict(x=P + 2), dict(y=P + 1), dict(n=P + 1), dict(gate=P + 1),
    dict(scale=P + 2), dict(pre=H.Norm(1, 1e-5, P + 1, None))], ids=str)
def test_norm_refusals(kw):
    refused(H.lib().bnh_block_norm(norm_args(**kw), 10, 64, 2, None), "bnh_block_norm")


@pytest.mark.parametrize("M,C,B", [(0, 64, 2), (10, 0, 2), (10, 64, 0), (-1, 64, 2), (10, 16385, 1),
                                   (1 << 20, 64, 1 << 12)])
def test_norm_sizes_refused(M, C, B):
    a = norm_args(ldf=1 << 15, ldx=1 << 15, ldy=1 << 15, ldn=1 << 15, ldg=1 << 15, y_ws=1 << 50, n_ws=1 << 50)
    refused(H.lib().bnh_block_norm(a, M, C, B, None), "bnh_block_norm")
    refused(H.lib().bnh_block_norm(None, 10, 64, 2, None), "bnh_block_norm")


def lora(x=P, x_ws=640, lda=64, M=10, B=2, w=P, ldw=64, N=32, K=64, bias=P, L=(4, 8, P, P, P), idx=P, act=0, out=P,
         out_ws=320, ldo=32, opad=0, res=None, ldr=0, ws=P, wb=1 << 20):
    e = H.Epi16(act, out, out_ws, ldo, 0, opad, res, 0, ldr)
    return H.lib().bnh_pw_lora(x, x_ws, lda, M, B, w, ldw, N, K, bias, H.Lora(*L) if L else None, idx, e, ws, wb, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(out=None), dict(M=0), dict(B=0), dict(N=0), dict(K=0), dict(lda=63), dict(ldw=63),
    dict(ldo=31), dict(out_ws=319), dict(act=3), dict(act=-1), dict(opad=1), dict(res=P, ldr=31), dict(idx=None),
    dict(L=(4, 0, P, P, P)), dict(L=(4, 257, P, P, P)), dict(L=(-1, 8, P, P, P)), dict(L=(4, 8, None, P, P)),
    dict(L=(4, 8, P, None, P)), dict(ws=None), dict(ws=P + 8), dict(wb=63), dict(x=P + 1), dict(w=P + 1), dict(out=P + 1),
    dict(bias=P + 2), dict(idx=P + 2), dict(L=(4, 8, P + 1, P, P)), dict(L=(4, 8, P, P, P + 2)), dict(M=1 << 20, B=1 << 12,
                                                                                                      out_ws=1 << 40)],
    ids=str)
def test_lora_refusals(kw):
    refused(lora(**kw), "bnh_pw_lora")


def test_lora_work_bytes():
    L = H.lib()
    assert L.bnh_pw_lora_work_bytes(10, 2, 32, 64, 8) > 0
    for bad in ((0, 2, 32, 64, 8), (10, 0, 32, 64, 8), (10, 2, 32, 64, 257), (10, 2, 32, 64, -1)):
        assert L.bnh_pw_lora_work_bytes(*bad) == 0
        assert b"check failed" in L.bnh_last_error()


def la_args(**kw):
    a = H.LinAttn(q=P, k=P, v=P, o=P, f16=1, ldq=64, ldk=64, ldv=96, ldo=96, H=4, Hq=4, Hk=4, Hv=4, dk=16, dv=24, g=P,
                  ldg=4, scale=1.0, s0=P, s1=P, slots=8, slot=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(g=None), dict(ldq=63), dict(ldk=63), dict(ldv=95),
    dict(ldo=95), dict(ldg=3), dict(H=0), dict(Hq=3), dict(Hk=0), dict(Hv=8), dict(dk=0), dict(dk=257), dict(dv=0),
    dict(dv=257), dict(f16=2), dict(slots=-1), dict(slot=None, slots=1), dict(q=P + 1), dict(o=P + 1), dict(g=P + 2),
    dict(s0=P + 2), dict(s1=P + 1), dict(slot=P + 2)], ids=str)
def test_la_refusals(kw):
    refused(H.lib().bnh_linattn(la_args(**kw), 5, 2, 10, P, P, P, 1 << 30, None))


@pytest.mark.parametrize("T,B,rows,start", [(0, 2, 10, P), (5, 0, 10, P), (5, 2, 0, P), (5, 2, 9, None),
                                            (1, 1 << 23, 1 << 24, P), ((1 << 30) + 1, 1, 10, P)])
def test_la_sizes_refused(T, B, rows, start):
    a = la_args(slots=1 << 24)
    refused(H.lib().bnh_linattn(a, T, B, rows, start, P, P, 1 << 30, None))


def test_la_work_bytes():
    L = H.lib()
    for bad in ((la_args(), 0, 2), (la_args(), 5, 0), (la_args(dk=257), 5, 2), (None, 5, 2)):
        assert L.bnh_linattn_work_bytes(*bad) == 0
        assert b"check failed" in L.bnh_last_error()
    # one long sequence is cut into pieces, and has to have the workspace that it is asked for
    a = la_args(dk=64, dv=64, ldq=256, ldk=256, ldv=256, ldo=256)
    need = L.bnh_linattn_work_bytes(a, 1 << 14, 1)
    if need:
        refused(L.bnh_linattn(a, 1 << 14, 1, 1 << 14, None, None, P, need - 1, None))
        refused(L.bnh_linattn(a, 1 << 14, 1, 1 << 14, None, None, None, need, None))
        refused(L.bnh_linattn(a, 1 << 14, 1, 1 << 14, None, None, P + 8, need, None))
