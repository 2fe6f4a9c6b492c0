"""How attention with sinks numbers the tokens that a tile sees (csrc/paged_plan.h,
compiled for the host): every seen token has one number, in steps of 64 that are
whole on either side of the hole, and the sinks before a hole lie in full pages."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from conftest import PKG

GLUE = """
#include "paged_plan.h"
using namespace qtts;
extern "C" void hole(int low, int high, int sinks, int *o) {
    const SeenHole h = seen_hole(low, high, sinks);
    o[0] = h.hole; o[1] = h.edge;
}
extern "C" long long span(int window, int sinks) { return seen_span(window, sinks); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("sinks")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.span.restype = C.c_longlong
    return lib


def test_numbers(lib):
    r = np.random.default_rng(1)
    out = (C.c_int * 2)()
    holes = 0
    for _ in range(3000):
        rows, page = int(r.integers(1, 33)), int(r.choice([16, 32, 64, 128]))
        start, window, sinks = int(r.integers(0, 1500)), int(r.integers(1, 400)), int(r.integers(1, 400))
        low, high, end = max(0, start - window + 1), start + rows, start + rows + int(r.integers(0, 40))
        lib.hole(low, high, sinks, out)
        hole, edge = out
        assert hole % 64 == 0 and edge % 64 == 0 and 0 <= hole <= high
        seen = {t for p in range(start, start + rows) for t in range(p + 1) if t > p - window or t < sinks}
        total = high - hole
        tokens = [v + (hole if v >= edge else 0) for v in range(total)]
        assert seen <= set(tokens) and len(set(tokens)) == total and max(tokens) < high
        assert total <= max(lib.span(window, sinks), high if not hole else 0)
        if hole:
            holes += 1
            full = end // page * page
            assert edge <= full and edge <= low // 64 * 64 - 64
            # the last number of a full page's token: what the steps stop at
            stop = max(edge, min(full, high) - hole)
            assert [t for t in tokens[:stop] if t >= full] == [] and [t for t in tokens[stop:] if t < min(full, high)] == []
    assert holes > 500
    lib.hole(0, 1 << 30, 2 ** 31 - 1, out)
    assert tuple(out) == (0, 1 << 30)
    assert lib.span(2 ** 31 - 1, 2 ** 31 - 1) > 2 ** 32 - 2
