"""Lists that the Python binding hands to the library: one entry per cache, 32 bits (CPU)."""
import numpy as np
import pytest

import eakv_amd as E


class Handle:
    def __init__(self, h):
        self.h = h


def test_window_plan_lengths():
    """The library reads n_tokens[i] and starts[i] of every cache."""
    caches = [Handle(None), Handle(None)]
    for n, starts in (([4], None), ([4, 4, 4], None), ([], None), ([4, 4], [0]), ([4, 4], [0, 0, 0]),
                      (np.array([4]), None)):
        with pytest.raises(ValueError):
            E.WindowPlan(caches, n, 8, 8, starts=starts)
    p = E.WindowPlan(caches, np.array([4, 3]), 8, 8, starts=(1, 2))
    assert list(p._n) == [4, 3] and list(p._starts) == [1, 2]


def test_values_beyond_32_bits():
    """A position of 2^32 + 5 is not position 5."""
    for x in (2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1):
        with pytest.raises(ValueError):
            E.ints([0, x])
    assert list(E.ints([2 ** 31 - 1, -2 ** 31, np.int64(7)])) == [2 ** 31 - 1, -2 ** 31, 7]
    cache = E.Cache(0, 0, 0, 0, _handle=1)
    try:
        with pytest.raises(ValueError):
            cache.compact(np.array([2 ** 32 + 5]))
    finally:
        cache.h = None
