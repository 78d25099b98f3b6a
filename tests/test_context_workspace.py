"""The workspace that linear attention asks for, on the host (the pointers are never read)."""
import pytest

from bnneon import hip as H
from test_context_refusals import P, la_args, refused


def args(f16, heads, d):
    return la_args(f16=f16, H=heads, Hq=heads, Hk=heads, Hv=heads, dk=d, dv=d, ldq=heads * d, ldk=heads * d,
                   ldv=heads * d, ldo=heads * d, ldg=heads, slots=1 << 20)


@pytest.mark.parametrize("f16,heads,d,T,B", [(1, 4, 64, 1 << 14, 1), (1, 12, 128, 720, 10), (0, 16, 64, 500, 8),
                                             (1, 1, 256, 300, 3)])
def test_short_workspace_refused(f16, heads, d, T, B):
    """Sequences that are cut into pieces need a workspace, and a call without all of it is refused."""
    L, a = H.lib(), args(f16, heads, d)
    need = L.bnh_linattn_work_bytes(a, T, B)
    # a state of each piece but the last and of the start at least, of two pieces or more
    assert need >= 2 * 4 * B * heads * d * d
    for work, size in ((P, need - 1), (None, need), (P + 8, need)):
        refused(L.bnh_linattn(a, T, B, T * B, None, None, work, size, None), "bnh_linattn")


def test_no_workspace():
    """The recurrence, and sequences of a few chunks, need none."""
    L = H.lib()
    for f16, heads, d, T, B in ((1, 12, 128, 1, 64), (1, 12, 128, 8, 1), (1, 12, 128, 256, 1), (0, 4, 64, 128, 1)):
        assert L.bnh_linattn_work_bytes(args(f16, heads, d), T, B) == 0
