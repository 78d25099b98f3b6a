"""What the temporal context net asks of the device, and in which order: against a library that only notes its calls."""
import itertools

import pytest

from bnneon import contextnet, hip


class Notes:
    """Entry points that do nothing and succeed; `calls` has their names and arguments."""

    def __init__(self):
        self.calls, self.at, self.fail = [], itertools.count(1 << 20, 1 << 20), None

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            if name == "bnh_malloc":
                return next(self.at)
            if name == "bnh_last_error":
                return b"refused"
            return 1 if name == self.fail else 0
        return call

    def names(self):
        return [n for n, _ in self.calls]


@pytest.fixture
def notes(monkeypatch):
    n = Notes()
    monkeypatch.setattr(hip, "lib", lambda: n)
    return n


def net(**kw):
    return contextnet.ContextNet(**{**dict(dim=64, heads=2, layers=2, stations=3, rank=2, cached=[1], windows=100, page=16), **kw})


@pytest.mark.parametrize("cached", [[], [0], [0, 1]])
@pytest.mark.parametrize("what", ["forget", "reset"])
def test_clearing_waits(notes, cached, what):
    """Runs on any stream are over before a station's states are cleared (which returns once it is done) and its pages are free."""
    x = net(cached=cached)
    p = x.plan([20, 1], [0, 2])
    x.run(p, stream=77)
    notes.calls.clear()
    x.forget(0) if what == "forget" else x.reset()
    names = notes.names()
    clears = [i for i, n in enumerate(names) if n == "bnh_memset"]
    assert names[0] == "bnh_device_sync"
    assert len(clears) == 2 - len(cached)


@pytest.mark.parametrize("entry", ["bnh_block_norm", "bnh_pw_lora", "bnh_kv_append", "bnh_kv_select", "bnh_kv_attn"])
def test_a_run_that_fails_does_not_move_the_caches(notes, entry):
    """A call that is refused leaves each station's windows where they were, and its next run puts its rows there; pages that it has
    been given stay its own."""
    x = net(seen=3)
    p, other = x.plan([20, 1], [0, 2]), x.plan([5], [1])
    x.run(p)
    x.run(other)
    past, pages = list(x.past), len(x.free)
    notes.fail = entry
    with pytest.raises(hip.HipError):
        x.run(p)
    assert list(x.past) == past == [20, 5, 1]
    assert len(x.free) == pages - 1  # the 33rd to 40th window's page
    notes.fail = None
    x.run(p)
    assert list(x.past) == [40, 5, 2] and len(x.free) == pages - 1
    assert sorted(x.free + [i for i in x.table.ravel() if i >= 0]) == list(range(x.pages))


@pytest.mark.parametrize("page", [16, 1024])
def test_as_many_windows_as_a_table_can_have(notes, page):
    """A station's tokens are numbered in 31 bits: what no call would take is refused when the net is made."""
    most = ((1 << 31) - 1024 - 1) // page * page
    for n in (most + 1, 1 << 31, 1 << 40):
        with pytest.raises(ValueError, match="windows"):
            net(windows=n, page=page, pages=8, cached=[0], stations=1)
        assert not notes.calls
    if page == 1024:
        x = net(windows=most, page=page, pages=8, cached=[0], stations=1)
        assert x.ldt * page < (1 << 31) - 1024
