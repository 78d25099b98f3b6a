"""The temporal context net with blocks over a cache of the stations' windows: archive and live calls against the same blocks in
64 bits, captured calls, and the pages that stations share."""
import ctypes

import numpy as np
import pytest

import cache_ref as K
import context_ref as R

pytestmark = pytest.mark.gpu


def reference(net, x, station):
    """One sequence's rows x [T][dim] from its first on through the blocks in float64."""
    d, T = net.dim // net.heads, len(x)
    x = x.astype(np.float64)

    def rms(u, w):
        return u / np.sqrt((u * u).mean(-1, keepdims=True) + 1e-6) * w

    def linear(h, u):
        w, a, b = (h[k].astype(np.float64) for k in ("w", "a", "b"))
        return u @ w.T + h["bias"] + (u @ a[station].T) @ b[station].T

    for i, h in enumerate(net.host):
        y = linear(h["win"], rms(x, h["pre"]))
        q, k, v, gate = (y[:, j * net.dim:(j + 1) * net.dim] for j in range(4))
        q, k, v = (z.reshape(T, net.heads, d) for z in (q, k, v))
        if i in net.cached:
            q, k = (K.rotate(z, np.arange(T), net.rd, 0, net.freq)[0] for z in (q, k))
            seen = np.repeat(np.tril(np.ones((T, T), bool))[:, None], net.heads, 1)
            o, _ = K.attention(q, k, v, seen, d ** -0.5, 0)
        else:
            o, *_ = R.linattn(q, k, v, np.repeat(net.g[None], T, 0), d ** -0.5, np.zeros((net.heads, d, d)))
        f = linear(h["wout"], o.reshape(T, net.dim))
        x = x + h["scale"] * R.act(gate, 1) * rms(f, h["post"])
    return x, rms(x, net.final)


def feed(hip, net, xs, calls):
    """Sequences through the net in calls of (lengths, stations), each from where its station's last call ended -> {station: x, n}"""
    at, got = {s: 0 for s in xs}, {s: ([], []) for s in xs}
    for lens, stations in calls:
        p = net.plan(lens, stations)
        p["x"].upload(np.concatenate([xs[s][at[s]:at[s] + n] for s, n in zip(stations, lens)]))
        net.run(p)
        hip.sync()
        x, n = p["x"].numpy(), p["n"].numpy()
        for s, m, e in zip(stations, lens, np.cumsum(lens)):
            got[s][0].append(x[e - m:e]), got[s][1].append(n[e - m:e])
            at[s] += m
    return {s: tuple(np.concatenate(z) for z in v) for s, v in got.items()}


CALLS = [([70, 1, 33, 130], [4, 0, 5, 2]), ([1, 1, 1, 1], [2, 4, 0, 5]), ([9, 40], [0, 4]), ([1, 0, 1, 1], [2, 0, 4, 5])]


@pytest.mark.parametrize("cached,seen,dim", [((1,), 0, 192), ((0, 1), 0, 192), ((0,), 64, 192), ((1,), 0, 99)])
def test_archive_then_live(hip, cached, seen, dim):
    """Calls of any lengths equal the whole sequences: within what rounding the blocks' rows to fp16 does (a few parts in 2^11
    each, over 2 blocks). 64 pages seen are all that there are."""
    from bnneon import contextnet
    net = contextnet.ContextNet(dim=dim, heads=3, layers=2, stations=6, rank=8, seed=3, cached=cached, windows=200, page=16, seen=seen)
    rng = np.random.default_rng(4)
    total = {s: 0 for s in (0, 2, 4, 5)}
    for lens, stations in CALLS:
        for n, s in zip(lens, stations):
            total[s] += n
    xs = {s: rng.standard_normal((n, dim)).astype(np.float32) for s, n in total.items()}
    got = feed(hip, net, xs, CALLS)
    for s, x in xs.items():
        for name, g, want in zip("xn", got[s], reference(net, x, s)):
            off = np.linalg.norm(g - want) / np.linalg.norm(want)
            print(f"station {s} {name}: {off:.2e}", flush=True)
            assert off < 8 * R.HU, (s, name, off)
    assert list(net.past) == [total.get(s, 0) for s in range(6)]
    assert len(net.free) + sum(-(-n // 16) for n in total.values()) == net.pages


def test_few_pages(hip):
    """With few pages seen, the windows that have no more than those look at all of them; the others give the same twice."""
    from bnneon import contextnet
    kw = dict(dim=128, heads=2, layers=1, stations=2, rank=4, seed=5, cached=[0], windows=400, page=16)
    x = np.random.default_rng(6).standard_normal((300, 128)).astype(np.float32)
    calls = [([200], [1]), ([1], [1]), ([99], [1])]
    few = [feed(hip, contextnet.ContextNet(**kw, seen=4), {1: x}, calls)[1] for _ in range(2)]
    every = feed(hip, contextnet.ContextNet(**kw), {1: x}, calls)[1]
    for a, b, c in zip(*few, every):
        assert np.array_equal(a, b) and np.isfinite(a).all()
        off = np.linalg.norm(a[:64] - c[:64]) / np.linalg.norm(c[:64])
        assert off < 8 * R.HU, off
        assert not np.array_equal(a[64:], c[64:])


def test_pages_run_out(hip):
    """A call that needs more pages or windows than there are is refused, and nothing has moved; pages come back."""
    from bnneon import contextnet
    net = contextnet.ContextNet(dim=64, heads=2, layers=1, stations=3, rank=2, cached=[0], windows=100, page=16, pages=7)
    rng = np.random.default_rng(1)

    def call(lens, stations):
        p = net.plan(lens, stations)
        p["x"].upload(rng.standard_normal((sum(lens), 64)).astype(np.float32))
        net.run(p)
        hip.sync()

    call([60], [0])
    with pytest.raises(ValueError, match="no pages"):
        call([30, 40], [0, 1])
    with pytest.raises(ValueError, match="more than"):
        call([41], [0])
    assert list(net.past) == [60, 0, 0] and len(net.free) == 3
    call([4, 40], [0, 1])
    assert not net.free
    net.forget(0)
    call([64], [2])
    assert list(net.past) == [0, 40, 64] and not net.free
    net.reset()
    assert len(net.free) == 7 and not net.past.any()


def test_a_station_starts_again(hip):
    """A forgotten station begins as in a new net, in the pages that came back; the other one goes on."""
    from bnneon import contextnet
    kw = dict(dim=96, heads=2, layers=2, stations=2, rank=4, seed=2, cached=[1], windows=64, page=16, pages=8)  # 4 pages a station of 60 windows
    rng = np.random.default_rng(3)
    x, y = rng.standard_normal((2, 60, 96)).astype(np.float32)
    net = contextnet.ContextNet(**kw)
    feed(hip, net, {0: x[:30], 1: y[:30]}, [([30, 30], [0, 1])])
    for wrong in (-1, 2):
        with pytest.raises(ValueError):
            net.forget(wrong)
    net.forget(0)
    got = feed(hip, net, {0: x, 1: y[30:]}, [([40, 30], [0, 1]), ([20], [0])])
    new = contextnet.ContextNet(**kw)
    for s, want in ((0, reference(new, x, 0)), (1, [z[30:] for z in reference(new, y, 1)])):
        for name, g, w in zip("xn", got[s], want):
            off = np.linalg.norm(g - w) / np.linalg.norm(w)
            assert off < 8 * R.HU, (s, name, off)


@pytest.mark.parametrize("seen", [0, 4])
def test_captured_in_a_graph(hip, seen):
    """A live call captured once and replayed between eager calls and synchronisations gives each time what the eager call gives
    from the same cache and rows."""
    from bnneon import contextnet
    hip.lib()
    rt = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    vp = ctypes.c_void_p

    def ok(rc):
        assert rc == 0, rc

    net = contextnet.ContextNet(dim=128, heads=2, layers=2, stations=5, rank=8, seed=7, cached=[1], windows=1500, page=16, seen=seen)
    rng = np.random.default_rng(8)
    first = rng.standard_normal((5 * 90, 128)).astype(np.float32)
    rows = [rng.standard_normal((5, net.dim)).astype(np.float32) for _ in range(4)]
    archive, p, other = net.plan([90] * 5, range(5)), net.plan([1] * 5, range(5)), None
    results = []
    for graphed in (False, True):
        net.reset()
        archive["x"].upload(first)
        net.run(archive)
        hip.sync()
        if graphed:
            stream, graph, call = hip.lib().bnh_stream_new(), vp(), vp()
            ok(rt.hipStreamBeginCapture(vp(stream), 0))
            net.run(p, stream, advance=False)
            ok(rt.hipStreamEndCapture(vp(stream), ctypes.byref(graph)))
            ok(rt.hipGraphInstantiate(ctypes.byref(call), graph, None, None, ctypes.c_size_t(0)))
            other = contextnet.ContextNet(dim=128, heads=2, layers=1, stations=1, rank=8, cached=[0], windows=100, page=16)
            q = other.plan([3], [0])
        got = []
        for x in rows:
            p["x"].upload(x)
            if graphed:
                net.advance(p, stream)
                ok(rt.hipGraphLaunch(call, vp(stream)))
                hip.sync(stream)
                q["x"].upload(x[:3])
                other.run(q)                             # eager work between the replays
                hip.sync()
            else:
                net.run(p)
                hip.sync()
            got.append((p["x"].numpy(), p["n"].numpy()))
        results.append(got)
    for a, b in zip(*results):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    ok(rt.hipGraphExecDestroy(call))
    ok(rt.hipGraphDestroy(graph))
    hip.check(hip.lib().bnh_stream_free(stream))
