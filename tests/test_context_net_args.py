"""What the temporal context net refuses when it is made, before anything is put on the device."""
import pytest

from bnneon import contextnet


@pytest.mark.parametrize("kw", [dict(dim=65, heads=2), dict(heads=0), dict(heads=-3), dict(dim=0), dict(dim=514, heads=2),
                                dict(dim=16640, heads=65), dict(layers=0), dict(stations=0), dict(rank=0), dict(rank=257)],
                         ids=str)
def test_refused(kw):
    with pytest.raises(ValueError):
        contextnet.ContextNet(**{**dict(dim=64, heads=2, layers=1, stations=2, rank=4), **kw})
