"""The temporal context net on streams that wait for nothing but themselves: stations that start again between runs."""
import numpy as np
import pytest

from test_gpu_context import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cached,seen", [((1,), 0), ((0, 1), 4), ((), 0)])
def test_a_station_starts_again_between_streams(hip, cached, seen):
    """A long run on one stream, the station forgotten at once, then runs on another stream, of a station that gets its pages and of
    itself: all as with a wait after each step."""
    from bnneon import contextnet
    say(f"streams cached {cached} seen {seen}")
    kw = dict(dim=256, heads=2, layers=2, stations=3, rank=4, seed=2, cached=cached, windows=2048, page=16, pages=300, seen=seen)
    x = np.random.default_rng(3).standard_normal((4, 2000, 256)).astype(np.float32)
    calls = [([2000, 40], [0, 2]), ([1900], [1]), ([300, 1], [0, 2])]
    results = []
    for patient in (True, False):
        net = contextnet.ContextNet(**kw)
        streams = [None] * 3 if patient else [hip.lib().bnh_stream_new() for _ in range(3)]
        plans = [net.plan(*c) for c in calls]
        for i, p in enumerate(plans):
            p["x"].upload(np.concatenate([x[i, :n] for n in p["lens"]]))
        net.run(plans[0], streams[0])
        if patient:
            hip.sync()
        net.forget(0)
        net.run(plans[1], streams[1])
        net.run(plans[2], streams[2])
        hip.device_sync()
        results.append([(p["x"].numpy(), p["n"].numpy()) for p in plans])
        net.reset()
        plans[2]["x"].upload(np.concatenate([x[2, :300], x[3, :1]]))
        net.run(plans[2], streams[0])
        hip.device_sync()
        results[-1].append((plans[2]["x"].numpy(), plans[2]["n"].numpy()))
        if not patient:
            for s in streams:
                hip.check(hip.lib().bnh_stream_free(s))
    for a, b in zip(*results):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    assert np.isfinite(results[0][0][0]).all()


def test_a_run_ahead_of_its_pages_stores_nothing(hip):
    """A run without advance() whose plan has been given no pages yet: no station's cache changes."""
    from bnneon import contextnet
    say("ahead of its pages")
    net = contextnet.ContextNet(dim=64, heads=2, layers=1, stations=3, rank=2, cached=[0], windows=100, page=16)
    x = np.random.default_rng(1).standard_normal((90, 64)).astype(np.float32)
    p = net.plan([30, 30, 30], range(3))
    p["x"].upload(x)
    net.run(p)
    hip.sync()
    before = [net.cache[0][k].numpy() for k in "kv"]
    other = net.plan([40, 50], [2, 0])
    other["x"].upload(x)
    net.run(other, advance=False)
    hip.sync()
    assert (other["table"].numpy() == -1).all() and not other["past"].numpy().any()
    for a, k in zip(before, "kv"):
        assert np.array_equal(a, net.cache[0][k].numpy())
    assert list(net.past) == [30, 30, 30]
