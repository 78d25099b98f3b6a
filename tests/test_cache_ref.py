"""What the definitions of the cached-attention operators give in cases that are worked out by hand."""
import numpy as np

import cache_ref as R


def test_forced_pages_come_before_infinite_scores():
    lo, hi = np.zeros((6, 1, 2), np.float32), np.ones((6, 1, 2), np.float32)
    hi[1:4] = np.inf
    q, there = np.ones((1, 2), np.float32), np.ones(6, bool)
    for first, last, n, want in ((1, 1, 2, [0, 5]), (1, 1, 3, [0, 1, 5]), (0, 2, 3, [1, 4, 5]), (0, 0, 2, [1, 2]), (2, 0, 3, [0, 1, 2])):
        assert R.select(q, lo, hi, there, 95, 16, 0, first, last, n)[0].tolist() == want
