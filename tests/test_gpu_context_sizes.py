"""The temporal context operators at sizes past what one launch may have threads for (2^32)."""
import numpy as np
import pytest

from test_gpu_context import say

pytestmark = pytest.mark.gpu


def part(H, ptr, n, dtype):
    """n values from a device address."""
    a = np.empty(n, dtype)
    H.check(H.lib().bnh_memcpy_d2h(a.ctypes.data, ptr, a.nbytes))
    return a


def test_norm_many_rows(hip):
    """2^28 + rows of one value, 16 threads each: windows that share their input."""
    H, M, B = hip, 1 << 14, (1 << 14) + 3
    say("norm many rows")
    x = np.linspace(-3, 3, M, dtype=np.float32).astype(np.float16)
    dx, y = H.DeviceArray.from_host(x), H.DeviceArray.zeros((B * M,), np.float16)
    a = H.BlockNorm(f16=1, x16=1, x=dx.ptr, x_ws=0, ldx=1, y=y.ptr, y_ws=M, ldy=1)
    H.check(H.lib().bnh_block_norm(a, M, 1, B, None), "block_norm")
    H.sync()
    assert (y.numpy().reshape(B, M) == x).all()


def test_adapters_many_rows(hip):
    """2^28 + rows, windows of two adapters and of none."""
    H, M, B, K, N, r = hip, 1 << 14, (1 << 14) + 3, 8, 8, 4
    say("adapters many rows")
    rng = np.random.default_rng(0)
    x = rng.integers(-4, 5, (M, K)).astype(np.float16)
    w, a = rng.integers(-3, 4, (N, K)).astype(np.float16), rng.integers(-2, 3, (2, r, K)).astype(np.float16)
    b = rng.integers(-2, 3, (2, N, r)).astype(np.float16)
    idx = (np.arange(B) % 3 - 1).astype(np.int32)
    dx, dw, da, db, di = (H.DeviceArray.from_host(z) for z in (x, w, a, b, idx))
    out = H.DeviceArray.zeros((B * M * N,), np.float16)
    wb = H.lib().bnh_pw_lora_work_bytes(M, B, N, K, r)
    ws = H.DeviceArray((wb,), np.uint8)
    H.check(H.lib().bnh_pw_lora(dx.ptr, 0, K, M, B, dw.ptr, K, N, K, None, H.Lora(2, r, da.ptr, db.ptr, None), di.ptr,
                                H.Epi16(0, out.ptr, M * N, N, 0, 0, None, 0, 0), ws.ptr, wb, None), "pw_lora")
    H.sync()
    f = [z.astype(np.float64) for z in (x, w, a, b)]
    want = [f[0] @ f[1].T] + [f[0] @ f[1].T + (f[0] @ f[2][j].T) @ f[3][j].T for j in range(2)]
    assert max(np.abs(z).max() for z in want) < 2048  # whole numbers: fp16 holds them, the first product has few
    for i in (0, 1, 2, 255, 256, 8191, 8192, B - 4, B - 3, B - 2, B - 1):
        got = part(H, out.ptr + 2 * i * M * N, M * N, np.float16).reshape(M, N)
        assert np.array_equal(got, want[idx[i] + 1]), i


def test_projection_most_rows(hip):
    """2^31 - 2 rows of one value each, tiles of 128."""
    H, M, B = hip, 42966, 49981
    say("projection most rows")
    x = (np.arange(M) % 1000).astype(np.float16)
    dx, dw = H.DeviceArray.from_host(x), H.DeviceArray.from_host(np.array([2], np.float16))
    out = H.DeviceArray.zeros((B * M,), np.float16)
    wb = H.lib().bnh_pw_lora_work_bytes(M, B, 1, 1, 0)
    assert wb == 0
    H.check(H.lib().bnh_pw_lora(dx.ptr, 0, 1, M, B, dw.ptr, 1, 1, 1, None, None, None,
                                H.Epi16(0, out.ptr, M, 1, 0, 0, None, 0, 0), None, 0, None), "pw_lora")
    H.sync()
    for i in (0, 1, B // 2, B - 2, B - 1):
        assert np.array_equal(part(H, out.ptr + 2 * i * M, M, np.float16), 2 * x), i


def test_linattn_many_states(hip):
    """More than 2^23 heads and sequences of two slices of columns each, a row a sequence."""
    H, heads, B, dv = hip, 1 << 16, 129, 129
    say("linattn many states")
    rng = np.random.default_rng(1)
    q, k, v = (rng.integers(-5, 6, (B, n)).astype(np.float16) for n in (1, 1, dv))
    dq, dk, dv_, g = (H.DeviceArray.from_host(z) for z in (q, k, v, np.zeros(heads, np.float32)))
    o = H.DeviceArray.zeros((B * heads * dv,), np.float16)
    a = H.LinAttn(q=dq.ptr, k=dk.ptr, v=dv_.ptr, o=o.ptr, f16=1, ldq=1, ldk=1, ldv=dv, ldo=heads * dv, H=heads, Hq=1, Hk=1,
                  Hv=1, dk=1, dv=dv, g=g.ptr, ldg=0, scale=1.0)
    H.check(H.lib().bnh_linattn(a, 1, B, B, None, None, None, 0, None), "linattn")
    H.sync()
    for i in (0, 1, 63, 64, B - 2, B - 1):
        got = part(H, o.ptr + 2 * i * heads * dv, heads * dv, np.float16).reshape(heads, dv)
        assert (got == q[i] * k[i] * v[i]).all(), i


def test_linattn_many_chunks(hip):
    """More than 2^23 blocks of chunks, most of them of sequences without a row."""
    H, heads, B, T, d = hip, 1 << 16, 129, 9, 65
    say("linattn many chunks")
    rng = np.random.default_rng(2)
    full = [0, 64, 127, 128]
    rows = T * len(full)
    lens, start = np.zeros(B, np.int32), np.zeros(B, np.int32)
    lens[full], start[full] = T, T * np.arange(len(full))
    q, k, v = (rng.integers(-3, 4, (rows, n)).astype(np.float16) for n in (1, 1, d))
    dq, dk, dv, ds, dl, g = (H.DeviceArray.from_host(z) for z in (q, k, v, start, lens, np.zeros(heads, np.float32)))
    o = H.DeviceArray.zeros((rows * heads * d,), np.float16)
    a = H.LinAttn(q=dq.ptr, k=dk.ptr, v=dv.ptr, o=o.ptr, f16=1, ldq=1, ldk=1, ldv=d, ldo=heads * d, H=heads, Hq=1, Hk=1,
                  Hv=1, dk=1, dv=d, g=g.ptr, ldg=0, scale=1.0)
    assert H.lib().bnh_linattn_work_bytes(a, T, B) == 0
    H.check(H.lib().bnh_linattn(a, T, B, rows, ds.ptr, dl.ptr, None, 0, None), "linattn")
    H.sync()
    got = o.numpy().reshape(rows, heads, d)
    for i in range(len(full)):
        s = slice(i * T, i * T + T)
        kv = (k[s].astype(np.float64) * v[s]).cumsum(0)
        want = q[s].astype(np.float64) * kv
        assert np.abs(want).max() < 2048 and (got[s] == want[:, None]).all(), i
