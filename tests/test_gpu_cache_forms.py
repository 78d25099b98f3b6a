"""Cached attention where its forms, cuts and launches change: widths by rows, many sequences in parts, captured calls that share a
workspace, other streams, and what two calls give."""
import ctypes

import numpy as np
import pytest

import cache_ref as R
from test_gpu_cache import ONE, TWO, Append, Attn
from test_gpu_context import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128), (256, 256), (200, 72), (126, 98), (62, 66), (200, 202),
                                   (127, 127), (24, 25), (1, 256)])
def test_rows_by_the_tile(hip, f16, page, dk, dv):
    """Rows for more than one block of the tiled form over many tiles, in one go and with gaps between pages and a window: pages
    within a tile and tiles within a page, rows aligned to 16 bytes, 4 and 2."""
    say(f"tile {dk} {dv} page {page} f16 {f16}")
    for window, gone in ((0, []), (90, [(0, 1), (0, 9), (1, 0)])):
        a = Attn(hip, [300, 3, 77], [150, 260, 2], 4, 2, dk, dv, page, f16, window=window, gone=gone, seed=dk + window)
        a.run()
        first = a.do.get()[0].copy()
        a.check(f"window {window}")
        a.run()
        assert np.array_equal(first, a.do.get()[0], equal_nan=True)


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("heads,hk,n", [(1, 1, 15), (1, 1, 16), (1, 1, 17), (4, 1, 4), (4, 1, 5), (1, 1, 32), (1, 1, 33), (8, 2, 16), (2, 2, 64),
                                        (2, 2, 65), (3, 1, 22)])
@pytest.mark.parametrize("d", [128, 256])
def test_rows_about_the_forms(hip, f16, heads, hk, n, d):
    say(f"rows {n} heads {heads} {hk} d {d} f16 {f16}")
    a = Attn(hip, [700, 0, 64], [n, n, 1], heads, hk, d, d, 64, f16, seed=n)
    a.run()
    a.check("rows")


@pytest.mark.parametrize("f16,d,heads,n", [(1, 64, 3, 605), (1, 128, 2, 257), (0, 64, 3, 300), (0, 256, 2, 25), (0, 128, 1, 33), (1, 256, 1, 17)])
@pytest.mark.parametrize("window", [300, 664, 1500, 2 ** 31 - 1])
def test_windows_in_parts(hip, f16, d, heads, n, window):
    """A window whose tokens are cut into parts: the last tile of rows has few of them, and looks at fewer tokens than the others."""
    say(f"window {window} rows {n} d {d} f16 {f16}")
    a = Attn(hip, [2000, 40, 1777], [n, n - 1, n // 2], heads, 1, d, d, 64, f16, window=window, seed=n)
    a.run()
    a.check("window")


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("n", [1, 40])
def test_many_sequences_in_parts(hip, f16, n):
    """More sequences than a wave has lanes, some of them long, most short, some without a row: cut into parts."""
    say(f"many sequences rows {n} f16 {f16}")
    B = 150
    lens = [n if i % 7 else 0 for i in range(B)]
    lens[0] = lens[77] = n
    pasts = [(i * 37) % 50 for i in range(B)]
    pasts[3], pasts[77], pasts[149] = 4000, 2500, 3000
    a = Attn(hip, pasts, lens, 1, 1, 64, 64, 64, f16, seed=n)
    a.run()
    a.check("many")


@pytest.mark.parametrize("f16", [0, 1])
def test_nobody(hip, f16):
    """Calls without a row that any sequence has leave everything as it was."""
    say(f"nobody f16 {f16}")
    for n in (1, 100):
        a = Attn(hip, [2000, 3], [n, n], 2, 2, 64, 64, 64, f16)
        a.c.dlen.upload(np.zeros(2, np.int32))
        a.run()
        assert (a.do.get()[0] == 7).all()


@pytest.mark.parametrize("sel", [False, True])
@pytest.mark.parametrize("n", [1, 50])
def test_workspace(hip, n, sel):
    """One byte fewer, or another alignment, is refused, and nothing has run."""
    say(f"workspace rows {n} {sel}")
    a = Attn(hip, [3000, 100], [n, n], 2, 2, 64, 64, 64, 1, sel=(lambda c: np.full((c.rows, 2, 60), -1)) if sel else None)
    L, c = hip.lib(), a.c
    wb = L.bnh_kv_attn_work_bytes(c.args(), a.args(), *c.seqs()[:3])
    if wb:
        ws = hip.DeviceArray(wb + 64, np.uint8)
        for p, b in ((ws.ptr, wb - 1), (ws.ptr + 8, wb), (None, wb)):
            assert L.bnh_kv_attn(c.args(), a.args(), *c.seqs(), p, b, None) != 0
    if sel:
        wb = L.bnh_kv_select_work_bytes(c.args(), a.args(), *c.seqs()[:3])
        ws = hip.DeviceArray(wb + 64, np.uint8)
        for p, b in ((ws.ptr, wb - 1), (ws.ptr + 8, wb), (None, wb)):
            assert wb == 0 or L.bnh_kv_select(c.args(), a.args(), 1, 2, *c.seqs(), p, b, None) != 0
    hip.sync()
    assert (a.do.get()[0] == 7).all()


def test_graphs_that_share_a_workspace(hip):
    """Dense calls of both forms and a selection with its attention, each captured into a graph of its own with one workspace for
    all, replayed in turn between eager calls and synchronisations on other rows and lengths: every replay gives what the eager
    call gives."""
    say("graphs")
    rt, vp, L = ctypes.CDLL("libamdhip64.so.7"), ctypes.c_void_p, hip.lib()

    def ok(rc):
        assert rc == 0, rc

    d, heads, hk, nsel = 64, 6, 2, 5
    calls = [Attn(hip, [3000, 9], [1, 1], heads, hk, d, d, 64, 1, seed=1), Attn(hip, [2500, 40], [60, 60], heads, hk, d, d, 16, 1, seed=2),
             Attn(hip, [1500, 700], [3, 3], heads, hk, d, d, 32, 1, seed=3, sel=lambda c: np.full((c.rows, hk, nsel), -1))]
    wb = 16
    for a in calls:
        wb = max(wb, L.bnh_kv_attn_work_bytes(a.c.args(), a.args(), *a.c.seqs()[:3]))
        if a.sel is not None:
            wb = max(wb, L.bnh_kv_select_work_bytes(a.c.args(), a.args(), *a.c.seqs()[:3]))
    ws, stream = hip.DeviceArray(wb, np.uint8), L.bnh_stream_new()

    def enqueue(a, s):
        if a.sel is not None:
            hip.check(L.bnh_kv_select(a.c.args(), a.args(), 1, 2, *a.c.seqs(), ws.ptr, wb, s))
        hip.check(L.bnh_kv_attn(a.c.args(), a.args(), *a.c.seqs(), ws.ptr, wb, s))

    graphs = []
    for a in calls:
        graph, call = vp(), vp()
        ok(rt.hipStreamBeginCapture(vp(stream), 0))
        enqueue(a, stream)
        ok(rt.hipStreamEndCapture(vp(stream), ctypes.byref(graph)))
        ok(rt.hipGraphInstantiate(ctypes.byref(call), graph, None, None, ctypes.c_size_t(0)))
        graphs.append((graph, call))
    rng = np.random.default_rng(9)
    for step in range(4):
        say(f"graphs replay {step}")
        want = []
        for a in calls:  # other queries, and a sequence that is shorter by some tokens
            a.dq.d.upload((rng.standard_normal(a.dq.d.shape)).astype(np.float16))
            a.c.dpast.upload(np.array([a.c.pasts[0] - 300 * step, a.c.pasts[1]], np.int32))
            a.do.d.fill(0)
            enqueue(a, None)
            hip.sync()
            want.append(a.do.d.numpy())
            assert np.isfinite(want[-1].astype(np.float32)).all()
            a.do.d.fill(0)
        for a, (_, call) in zip(calls, graphs):
            ok(rt.hipGraphLaunch(call, vp(stream)))
        hip.sync(stream)
        for a, w in zip(calls, want):
            assert np.array_equal(a.do.d.numpy(), w), step
    for graph, call in graphs:
        ok(rt.hipGraphExecDestroy(call))
        ok(rt.hipGraphDestroy(graph))
    hip.check(L.bnh_stream_free(stream))


@pytest.mark.parametrize("n", [1, 80])
def test_two_streams(hip, n):
    """Calls on two streams at once, each with a workspace of its own."""
    say(f"two streams rows {n}")
    L = hip.lib()
    calls = [Attn(hip, [2000, 40 + i], [n, n], 4, 2, 64, 64, 32, 1, seed=i) for i in range(2)]
    wb = max(L.bnh_kv_attn_work_bytes(a.c.args(), a.args(), *a.c.seqs()[:3]) for a in calls)
    ws, streams = [hip.DeviceArray(max(wb, 16), np.uint8) for _ in calls], [L.bnh_stream_new() for _ in calls]
    for _ in range(5):
        for a, w, s in zip(calls, ws, streams):
            hip.check(L.bnh_kv_attn(a.c.args(), a.args(), *a.c.seqs(), w.ptr, wb, s))
    for a, s in zip(calls, streams):
        hip.sync(s)
        a.check("stream")
        hip.check(L.bnh_stream_free(s))


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dk,dv,rd,pairs", [(108, 211, 108, 0), (40, 33, 24, 1), (44, 70, 20, 0), (24, 25, 8, 1), (24, 24, 8, 0), (200, 3, 40, 0),
                                            (12, 9, 0, 0), (64, 63, 64, 0), (64, 63, 32, 1), (4, 16, 4, 0)])
@pytest.mark.parametrize("pad,at,extra", [(0, 0, 0), (4, 4, 4), (2, 2, 2), (8, 1, 8), (1, 0, 8)])
def test_append_some_at_a_time(hip, f16, dk, dv, rd, pairs, pad, at, extra):
    """Widths, strides and places that allow 8, 4, 2 values of a row at a time, or one."""
    say(f"append {dk} {dv} rd {rd} pairs {pairs} pad {pad} at {at} f16 {f16}")
    a = Append(hip, [0, 40, 31, 7], [70, 1, 33, 0], 6, 2, dk, dv, rd, pairs, 32, f16, seed=dk + rd, pad=pad, at=at, extra=extra)
    a.run()
    a.check("some")


@pytest.mark.parametrize("f16", [0, 1])
def test_append_again(hip, f16):
    """The same rows once more at the same place change nothing, bounds neither: a call that failed half-way is made again."""
    say(f"append again f16 {f16}")
    a = Append(hip, [40, 7], [30, 21], 4, 2, 64, 48, 64, 0, 16, f16, seed=2)
    a.run()
    a.check("once")
    a.run()
    a.check("twice")


def test_weights_in_two_parts(hip):
    """A single fp16 row's weights are factors of 22 bits, many rows' of 11."""
    say("two parts")
    a = Attn(hip, [900, 33], [1, 1], 12, 4, 128, 128, 32, 1, seed=7)
    a.run()
    a.check("one row", TWO)
    a = Attn(hip, [900, 33], [6, 6], 12, 4, 128, 128, 32, 1, seed=7)
    a.run()
    a.check("rows", ONE)
    assert R.HU == 2.0 ** -11
