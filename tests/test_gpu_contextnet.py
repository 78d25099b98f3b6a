"""The temporal context net (bnneon.contextnet): archive and live calls against the same blocks in 64 bits, and over the
embeddings that a net of the engine leaves on the device."""
import ctypes

import numpy as np
import pytest

import context_ref as R

pytestmark = pytest.mark.gpu


def reference(net, x, station, states):
    """One sequence's rows x [T][dim] through the blocks in float64; states [layer][H][d][d] are replaced."""
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
        o, states[i], *_ = R.linattn(q, k, v, np.repeat(net.g[None], T, 0), d ** -0.5, states[i])
        f = linear(h["wout"], o.reshape(T, net.dim))
        x = x + h["scale"] * R.act(gate, 1) * rms(f, h["post"])
    return x, rms(x, net.final)


def test_archive_then_live(hip):
    """Sequences of several lengths at once, then their next windows one by one, equal the whole sequences: within what
    rounding the blocks' rows to fp16 does (a few parts in 2^11 each, over 2 blocks)."""
    from bnneon import contextnet
    net = contextnet.ContextNet(dim=192, heads=3, layers=2, stations=6, rank=8, seed=3)
    rng = np.random.default_rng(4)
    lens, stations, more = [70, 1, 33, 129], [4, 0, 5, 2], 3
    xs = [rng.standard_normal((n + more, net.dim)).astype(np.float32) for n in lens]
    p = net.plan(lens, stations)
    p["x"].upload(np.concatenate([x[:n] for x, n in zip(xs, lens)]))
    net.run(p)
    hip.sync()
    got_x = np.split(p["x"].numpy(), np.cumsum(lens)[:-1])
    got_n = np.split(p["n"].numpy(), np.cumsum(lens)[:-1])
    live = net.plan([1] * len(lens), stations)
    for t in range(more):
        live["x"].upload(np.stack([x[n + t] for x, n in zip(xs, lens)]))
        net.run(live)
        hip.sync()
        lx, ln = live["x"].numpy(), live["n"].numpy()
        got_x = [np.concatenate([a, lx[i:i + 1]]) for i, a in enumerate(got_x)]
        got_n = [np.concatenate([a, ln[i:i + 1]]) for i, a in enumerate(got_n)]
    d = net.dim // net.heads
    for i, (x, s) in enumerate(zip(xs, stations)):
        states = [np.zeros((net.heads, d, d)) for _ in range(net.layers)]
        wx, wn = reference(net, x, s, states)
        for name, got, want in (("x", got_x[i], wx), ("n", got_n[i], wn)):
            off = np.linalg.norm(got - want) / np.linalg.norm(want)
            print(f"sequence {i} {name}: {off:.2e}", flush=True)
            assert off < 8 * R.HU, (i, name, off)
        for layer in range(net.layers):
            got = net.state[layer].numpy()[s]
            off = np.linalg.norm(got - states[layer]) / np.linalg.norm(states[layer])
            assert off < 8 * R.HU, (i, layer, off)
    assert not net.state[0].numpy()[[1, 3]].any(), "a station of no sequence moved"


def test_over_the_engines_embeddings(hip, tmp_path):
    """Windows through a net of the engine, whose embeddings stay on the device, into the context net."""
    from bnneon import binding, contextnet, v24net
    path = str(tmp_path / "v24.bnpk")
    v24net.V24Net(seed=1, n_blocks=3).write(path)
    rng = np.random.default_rng(5)
    n = 6
    pcm = np.stack([v24net.signal(rng) for _ in range(n)]).astype(np.float32)
    with binding.Model(path) as m:
        net = contextnet.ContextNet(dim=m.info.emb_dim, heads=8, layers=1, stations=2, rank=4, seed=6)
        p = net.plan([4, 2], [1, 0])
        dp, do = hip.DeviceArray.from_host(pcm), hip.DeviceArray.zeros((n, m.info.n_classes), np.float32)
        st = np.zeros(n, np.int32)
        assert m.L.bnn_infer_batch_device(m.ctx, dp.ptr, n, do.ptr, p["x"].ptr, st.ctypes.data_as(binding._IP), None) == 0
        hip.sync()
        emb = p["x"].numpy()
        assert np.isfinite(emb).all() and emb.std() > 0
        net.run(p)
        hip.sync()
        got = p["x"].numpy()
    for rows, s in ((slice(0, 4), 1), (slice(4, 6), 0)):
        want, _ = reference(net, emb[rows], s, [np.zeros((8, net.dim // 8, net.dim // 8))])
        off = np.linalg.norm(got[rows] - want) / np.linalg.norm(want)
        print(f"station {s}: {off:.2e}", flush=True)
        assert off < 8 * R.HU


def test_plans_refused(hip):
    from bnneon import contextnet
    net = contextnet.ContextNet(dim=64, heads=2, layers=1, stations=3, rank=2)
    for lens, stations in (([1], [3]), ([1], [-1]), ([1, 1], [0, 0]), ([1], [0, 1]), ([], []), ([0], [0]), ([-1, 2], [0, 1])):
        with pytest.raises(ValueError):
            net.plan(lens, stations)
    with pytest.raises(ValueError):
        contextnet.ContextNet(dim=65, heads=2)


def test_captured_in_a_graph(hip):
    """A live call captured once and replayed between eager calls and synchronisations gives each time what the eager call
    gives from the same state and rows."""
    from bnneon import contextnet
    hip.lib()
    rt = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    vp = ctypes.c_void_p

    def ok(rc):
        assert rc == 0, rc

    net = contextnet.ContextNet(dim=128, heads=2, layers=2, stations=5, rank=8, seed=7)
    rng = np.random.default_rng(8)
    p = net.plan([1] * 5, range(5))
    rows = [rng.standard_normal((5, net.dim)).astype(np.float32) for _ in range(4)]
    want = []
    for x in rows:
        p["x"].upload(x)
        net.run(p)
        hip.sync()
        want.append((p["x"].numpy(), p["n"].numpy()))
    last = [s.numpy() for s in net.state]
    net.reset()
    stream, graph, call = hip.lib().bnh_stream_new(), vp(), vp()
    ok(rt.hipStreamBeginCapture(vp(stream), 0))
    net.run(p, stream)
    ok(rt.hipStreamEndCapture(vp(stream), ctypes.byref(graph)))
    ok(rt.hipGraphInstantiate(ctypes.byref(call), graph, None, None, ctypes.c_size_t(0)))
    other = net.plan([3], [0])
    for x, (wx, wn) in zip(rows, want):
        p["x"].upload(x)
        ok(rt.hipGraphLaunch(call, vp(stream)))
        hip.sync(stream)
        assert np.array_equal(p["x"].numpy(), wx) and np.array_equal(p["n"].numpy(), wn)
        kept = [z.numpy() for z in net.state]
        other["x"].upload(x[:3])
        net.run(other)                               # eager work between the replays
        hip.sync()
        for z, k in zip(net.state, kept):
            z.upload(k)
    for z, k in zip(net.state, last):
        assert np.array_equal(z.numpy(), k)
    ok(rt.hipGraphExecDestroy(call))
    ok(rt.hipGraphDestroy(graph))
    hip.check(hip.lib().bnh_stream_free(stream))
