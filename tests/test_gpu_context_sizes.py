"""The temporal context operators at sizes past what one launch may have threads for (2^32)."""
import numpy as np
import pytest

from test_gpu_context import say

pytestmark = pytest.mark.gpu


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
