"""The factors between the units that a tile's sums are held in (csrc/fp8_plan.h,
compiled for the host), in exact fractions: however often the unit changes, the
factors' product stays by the units' quotient.

Within 16 changes what is carried is at most half a place of a quotient, 2^-24 of it,
and from 16 to 16 as much again: 2^-23, and 2^-22 between any two blocks.  The tests
allow a thousandth of that for what is carried in whole 2^-48 by reciprocals that are
not exact."""
import ctypes as C
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

from conftest import PKG

GLUE = """
#include <cstring>
#include "fp8_plan.h"
using namespace qtts;
extern "C" unsigned unit(unsigned s) { return fp8_unit(s); }
extern "C" unsigned power(unsigned s) { return fp8_power(s); }
// The factors of n units, as the kernel has them: 16 blocks a row, 4 rows a wave.
extern "C" void factors(const float *unit, const float *inverse, int n, int *out) {
    int carried = 0;
    for (int b0 = 0; b0 < n; b0 += 16) {
        Fp8Change c[16];
        int before = 0, apart = -1;
        bool any = carried != 0;
        for (int i = 0; i < 16; i++) {
            const int b = b0 + i < n ? b0 + i : n - 1, a = b > 0 ? b - 1 : 0;
            c[i] = fp8_change(unit[a], unit[b], inverse[a], inverse[b]);
            if (b0 + i < n) out[b] = c[i].quotient + fp8_step(c[i], before);
            before = fp8_carry(c[i], before);
            if (fp8_apart(c[i].quotient)) apart = i;
        }
        carried += before;
        if (apart < 0) continue;
        const Fp8Change all{0, 0, c[apart].half};
        if (b0 + apart < n) out[b0 + apart] += fp8_step(all, carried);
        carried = fp8_carry(all, carried);
    }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("units")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wno-unused-variable", "-Wno-unused-but-set-variable", "-shared",
                    "-fPIC", "-I", os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.unit.restype = lib.power.restype = C.c_uint
    return lib


def _bits(x):
    return int(np.float32(x).view(np.uint32))


def _factors(lib, units, seed):
    """With reciprocals that are off by a step to either side."""
    units = np.ascontiguousarray(units, np.float32)
    inverse = np.float32(1) / units
    step = np.random.default_rng(seed).integers(-1, 2, units.size).astype(np.int32)
    inverse = (inverse.view(np.int32) + step).view(np.float32)
    out = np.zeros(units.size, np.int32)
    lib.factors(C.c_void_p(units.ctypes.data), C.c_void_p(inverse.ctypes.data), units.size, C.c_void_p(out.ctypes.data))
    return units, out.view(np.float32)


def _pattern(kind, n, seed):
    r = np.random.default_rng(seed)
    u = 1 + r.random(n)
    if kind == "alternating":
        u[::2], u[1::2] = u[0], u[-1]
    elif kind == "every sixteenth equal":
        u = np.resize(1 + r.random(15), n)
        u[15::16] = u[14::16][:u[15::16].size]
        for i in range(15, n, 16):
            u[i] = u[i - 1]
    elif kind == "signs":
        u *= np.where(r.random(n) < 0.5, 1, -1)
    elif kind == "by one place":
        u = 1 + 0.3 * r.random() + np.arange(n) % 3 * 2.0 ** -23
    elif kind == "around one":
        u = 1 + np.arange(n) % 3 * 2.0 ** -23
    elif kind == "few":
        u = r.choice([1.0, 1.5, 1 + 1 / 3, 1.9999999], n)
    return u


@pytest.mark.parametrize("kind", ["any", "alternating", "every sixteenth equal", "signs", "by one place", "around one", "few"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 48, 300, 1024])
def test_the_factors_product_stays(lib, kind, n):
    for seed in range(3 if n > 100 else 20):
        units, factors = _factors(lib, _pattern(kind, n, seed), seed)
        assert factors[0] == 1
        product, off = Fraction(1), []
        for u, f in zip(units, factors):
            product *= Fraction(float(f))
            off.append(float(product * Fraction(float(u)) / Fraction(float(units[0])) - 1))
        off = np.array(off)
        assert np.abs(off).max() <= 2.0 ** -23 * 1.001
        assert off.max() - off.min() <= 2.0 ** -22 * 1.001


def test_equal_units_change_nothing(lib):
    for seed in range(200):
        u = np.float32(1 + np.random.default_rng(seed).random())
        _, factors = _factors(lib, np.full(50, u), seed)
        assert np.all(factors == 1)


def test_scales(lib):
    for s in (1.5, -3e-5, 2.0 ** -117, 1.9 * 2.0 ** 117, 1e30):
        u = np.uint32(lib.unit(_bits(s))).view(np.float32)
        p = np.uint32(lib.power(_bits(s))).view(np.float32)
        assert 1 <= abs(u) < 2 and float(u) * float(p) == float(np.float32(s))
    for s, flags in ((0.0, 1), (-0.0, 1), (2.0 ** -118, 5), (1e-45, 5), (-(2.0 ** 118), 5), (3e38, 5), (np.inf, 2),
                     (-np.inf, 2), (np.nan, 2)):
        assert lib.unit(_bits(s)) == _bits(1) and lib.power(_bits(s)) & 7 == flags
