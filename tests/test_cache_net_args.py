"""What the temporal context net refuses of its cache, before anything is put on the device."""
import pytest

from bnneon import contextnet


@pytest.mark.parametrize("kw", [dict(cached=[2]), dict(cached=[-1]), dict(cached=[0], windows=0), dict(cached=[0], page=8),
                                dict(cached=[0], page=48), dict(cached=[0], page=2048), dict(cached=[0], pages=0),
                                dict(cached=[0], seen=2), dict(cached=[0], seen=-1), dict(cached=[0], seen=(1 << 20) + 1)], ids=str)
def test_refused(kw):
    with pytest.raises(ValueError):
        contextnet.ContextNet(**{**dict(dim=64, heads=2, layers=2, stations=2, rank=4), **kw})
