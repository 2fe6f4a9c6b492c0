"""The bound that attention's plan takes for what a tile sees with sinks
(csrc/paged_plan.h), held wherever sinks and window lie: apart, with a hole between
them, or met, where a tile counts from token 0."""
import ctypes as C

import numpy as np

from test_paged_sinks_plan import lib  # noqa: F401 (a fixture)


def test_a_tile_never_sees_more_than_the_plan_has(lib):  # noqa: F811
    r = np.random.default_rng(2)
    out = (C.c_int * 2)()
    met = apart = 0
    for _ in range(20000):
        rows = int(r.integers(1, 33))
        start, window, sinks = int(r.integers(0, 3000)), int(r.integers(1, 900)), int(r.integers(1, 900))
        low, high = max(0, start - window + 1), start + rows
        lib.hole(low, high, sinks, out)
        assert high - out[0] <= lib.span(window, sinks)
        met, apart = met + (out[0] == 0), apart + (out[0] > 0)
    assert met > 4000 and apart > 4000
    for page in range(0, 700, 64):  # at the borders of 64
        for d in range(-2, 3):
            for sinks in (1, 63, 64, 65, 128):
                for window in (1, 63, 64, 65, 400):
                    start = max(page + sinks + window + d, 0)
                    for rows in (1, 32):
                        lib.hole(max(0, start - window + 1), start + rows, sinks, out)
                        assert start + rows - out[0] <= lib.span(window, sinks)
