"""How calls of attention over a cache are cut, on the host."""
import pytest

from bnneon import hip as H
from test_cache_refusals import attn, cache


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("T,d", [(1, 128), (1, 256), (40, 128), (300, 64), (300, 256)])
def test_windows_wider_than_any_cache(f16, T, d):
    """A window up to the largest number cuts a call as none does."""
    c = cache(f16=f16, page=64, Hk=12, dk=d, dv=d, k_ps=12 * 64 * d, v_ps=12 * 64 * d, ldt=271)
    need = [H.lib().bnh_kv_attn_work_bytes(c, attn(H=12, ldq=12 * d, ldo=12 * d, window=w), T, 1, T)
            for w in (0, 1 << 20, 2 ** 31 - 1000, 2 ** 31 - 17, 2 ** 31 - 16, 2 ** 31 - 1)]
    assert need[0] > 0 and len(set(need)) == 1, need
