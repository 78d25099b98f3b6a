"""Cached attention and appending with more sequences than one launch has threads for."""
import numpy as np
import pytest

from test_gpu_context import say

pytestmark = pytest.mark.gpu


def cache(hip, B, hk, pages, seed):
    """One page of `pages` tokens that every sequence begins with, empty so far; values of head g are g + 1."""
    k = np.random.default_rng(seed).standard_normal((hk, pages)).astype(np.float16)
    v = np.repeat(np.arange(1, hk + 1, dtype=np.float16)[:, None], pages, 1)
    keep = [hip.DeviceArray.from_host(k), hip.DeviceArray.from_host(v), hip.DeviceArray.zeros((B,), np.int32),
            hip.DeviceArray.zeros((B,), np.int32)]
    c = hip.KvCache(k=keep[0].ptr, v=keep[1].ptr, k_ps=hk * pages, v_ps=hk * pages, f16=1, pages=1, page=pages, Hk=hk, dk=1, dv=1,
                    table=keep[2].ptr, ldt=1, past=keep[3].ptr)
    return c, keep


@pytest.mark.parametrize("T,B,hk", [(1, (1 << 22) + 5, 3), (17, (1 << 18) + 3, 17)])
def test_attention_of_more_sequences_than_a_launch_takes(hip, T, B, hk):
    """2^23 blocks of 256 threads and more, and 2^22 of 512 in the tiled form: every row of the last sequences too."""
    say(f"attention of {B} sequences of {T} rows")
    L, rows = hip.lib(), T * B
    c, keep = cache(hip, B, hk, 32, T)
    q, o = hip.DeviceArray.zeros((rows, hk), np.float16), hip.DeviceArray((rows, hk), np.float16)
    o.fill(0x7f)
    a = hip.KvAttn(q=q.ptr, ldq=hk, o=o.ptr, ldo=hk, H=hk, scale=1.0, window=0)
    assert L.bnh_kv_attn_work_bytes(c, a, T, B, rows) == 0
    hip.check(L.bnh_kv_attn(c, a, T, B, rows, None, None, None, 0, None))
    hip.sync()
    assert (o.numpy() == np.arange(1, hk + 1)).all()


def test_append_of_more_sequences_than_a_launch_takes(hip):
    say("append of many sequences")
    L, B, hk = hip.lib(), (1 << 22) + 5, 3
    c, keep = cache(hip, B, hk, 16, 2)
    keep[2].fill(0xff)  # no pages: queries alone
    x = (np.arange(B * hk) % 2039).astype(np.float16).reshape(B, hk)
    q, qr = hip.DeviceArray.from_host(x), hip.DeviceArray((B, hk), np.float16)
    qr.fill(0x7f)
    hip.check(L.bnh_kv_append(c, None, q.ptr, hk, q.ptr, hk, q.ptr, hk, qr.ptr, hk, hk, 1, B, B, None, None, None))
    hip.sync()
    assert np.array_equal(qr.numpy(), x)
    # and a page each
    pool = [hip.DeviceArray.zeros((B, hk, 16), np.float16) for _ in range(2)]
    keep[2].upload(np.arange(B, dtype=np.int32)[::-1])
    c.k, c.v, c.pages = pool[0].ptr, pool[1].ptr, B
    hip.check(L.bnh_kv_append(c, None, q.ptr, hk, q.ptr, hk, None, 0, None, 0, hk, 1, B, B, None, None, None))
    hip.sync()
    for p in pool:
        got = p.numpy()
        assert np.array_equal(got[::-1, :, 0], x) and not got[..., 1:].any()
