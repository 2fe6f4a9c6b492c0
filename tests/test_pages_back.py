"""Which pages a row has after going back (csrc/pages_plan.h, compiled for the host):
dropped ones do not return, and what has to be asked for so that none is missed."""
import numpy as np

from test_pages_plan import lib  # noqa: F401 (a fixture)


def _seen(j, tokens, page, window, sinks):
    """Whether the next row of attention sees a token of a full page or of the one begun."""
    return j * page < tokens and any(t > tokens - window or t < sinks
                                     for t in range(j * page, min((j + 1) * page, tokens)))


def test_a_window_wider_by_what_a_row_goes_back(lib):  # noqa: F811
    r = np.random.default_rng(4)
    missed = 0
    for _ in range(3000):
        page = int(r.choice([16, 32, 64, 128]))
        window, sinks, back = int(r.integers(1, 300)), int(r.integers(0, 100)), int(r.integers(1, 200))
        tokens = int(r.integers(back, 900))
        then = tokens - int(r.integers(0, back + 1))
        for j in range(tokens // page + 1):
            if _seen(j, then, page, window, sinks):
                assert lib.kept(j, tokens, 1, page, window + back, sinks)
                missed += not lib.kept(j, tokens, 1, page, window, sinks)
    assert missed > 300  # with attention's own window
    # pages of 16, a window of 100: back from 1000 tokens to 992 needs token 893
    assert _seen(55, 992, 16, 100, 0) and not lib.kept(55, 1000, 1, 16, 100, 0) and lib.kept(55, 1000, 1, 16, 108, 0)
