"""The checks and the division of products on 8-bit floats (csrc/fp8_plan.h),
compiled for the host, and the oracle of their GPU tests against itself."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import fp8_model as fm
import qtts
from conftest import PKG

GLUE = """
#include "fp8_plan.h"
using namespace qtts;
static const char *why;
static int told(const Refusal &r) { why = r.why; return r.status; }
extern "C" const char *reason() { return why ? why : ""; }
extern "C" int gemm(const qtts_fp8_weight *w, const float *x, int ld_x, int rows, const float *add, int ld_add,
                    const float *y, int ld_y) {
    return told(check_fp8_gemm(*w, x, ld_x, rows, add, ld_add, y, ld_y));
}
extern "C" int quantize(const float *src, int ld, const qtts_fp8_weight *w) { return told(check_fp8_quantize(src, ld, *w)); }
extern "C" int own(int rows, int n, int kb) { return fp8_own_rows(rows, n, kb) ? (int)fp8_own_bytes(rows, kb) : 0; }
extern "C" void plan(int rows, int n, int k, long long *o) {
    const Fp8Plan p = fp8_plan(rows, n, k);
    o[0] = p.bn; o[1] = p.bm; o[2] = p.tiles_n; o[3] = p.tiles_m; o[4] = p.splits;
    o[5] = fp8_rows_at_once(k); o[6] = kFp8PartFloats; o[7] = kFp8MaxSplits; o[8] = kFp8RowStep;
    o[9] = (long long)kFp8ScratchBytes; o[10] = fp8_blocks(k); o[11] = p.waves; o[12] = p.each; o[13] = p.whole;
    o[14] = fp8_launched(p);
}
"""

OK, EINVAL, ESHAPE, ERANGE = qtts.QTTS_OK, qtts.QTTS_EINVAL, qtts.QTTS_ESHAPE, qtts.QTTS_ERANGE
AT = 1 << 20  # an address that is never read


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp8")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.reason.restype = C.c_char_p
    lib.gemm.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_int]
    lib.quantize.argtypes = [C.c_void_p, C.c_int, C.c_void_p]
    return lib


def _weight(**over):
    v = dict(codes=AT, scales=AT, n=300, k=272, ld=272)
    v.update(over)
    return qtts.Fp8Weight(*v.values())


@pytest.mark.parametrize("weight,status", [
    (dict(), OK), (dict(n=1), OK), (dict(n=1 << 17), OK), (dict(n=0), ESHAPE), (dict(n=(1 << 17) + 1), ESHAPE),
    (dict(k=16), OK), (dict(k=0), ESHAPE), (dict(k=264), ESHAPE), (dict(k=288), ESHAPE), (dict(ld=256), ESHAPE),
    (dict(ld=280), EINVAL), (dict(ld=288), OK), (dict(ld=1 << 23), OK), (dict(ld=(1 << 23) + 16), ERANGE), (dict(codes=0), EINVAL), (dict(scales=0), EINVAL),
    (dict(codes=AT + 8), EINVAL), (dict(scales=AT + 2), EINVAL), (dict(n=-5), ESHAPE),
])
def test_weights(lib, weight, status):
    w = C.byref(_weight(**weight))
    assert lib.gemm(w, AT, 1 << 17, 3, None, 0, AT + 64, 1 << 17) == status, lib.reason()
    assert lib.quantize(AT, 1 << 17, w) == status
    assert bool(lib.reason()) == (status != OK)


@pytest.mark.parametrize("args,status", [
    ((AT, 272, 3, None, 0, AT + 64, 300), OK), ((None, 0, 0, None, 0, None, 0), OK),
    ((AT, 272, -1, None, 0, AT + 64, 300), ESHAPE), ((AT, 272, (1 << 24) + 1, None, 0, AT + 64, 300), ESHAPE),
    ((None, 272, 3, None, 0, AT, 300), EINVAL), ((AT, 272, 3, None, 0, None, 300), EINVAL),
    ((AT, 268, 3, None, 0, AT + 64, 300), ESHAPE), ((AT, 272, 3, None, 0, AT + 64, 296), ESHAPE),
    ((AT, 274, 3, None, 0, AT + 64, 300), EINVAL), ((AT + 4, 272, 3, None, 0, AT + 64, 300), EINVAL),
    ((AT, 272, 3, None, 0, AT + 8, 300), EINVAL), ((AT, 300, 3, None, 0, AT, 300), EINVAL),
    ((AT, 272, 3, AT + 64, 300, AT + 64, 300), OK), ((AT, 272, 3, AT + 64, 304, AT + 64, 300), EINVAL),
    ((AT, 272, 3, AT + 640, 304, AT + 64, 300), OK), ((AT, 272, 3, AT + 640, 296, AT + 64, 300), ESHAPE),
    ((AT, 272, 3, AT + 4, 300, AT + 64, 300), EINVAL),
])
def test_rows(lib, args, status):
    assert lib.gemm(C.byref(_weight()), *args) == status, lib.reason()


def test_sources(lib):
    w = C.byref(_weight())
    assert lib.quantize(AT, 272, w) == OK
    assert lib.quantize(None, 272, w) == EINVAL
    assert lib.quantize(AT + 4, 272, w) == EINVAL
    assert lib.quantize(AT, 268, w) == ESHAPE


def test_plans(lib):
    """Tiles cover the output, splits the contraction, none of them empty; parts
    and the rows' scratch hold what a launch uses."""
    o = (C.c_longlong * 15)()
    for rows in [*range(1, 300, 7), 512, 1064, 4096, 8192, 100000, 1 << 24]:
        for n in (1, 31, 128, 1000, 2048, 12288, 131072):
            for k in (16, 128, 144, 2048, 6144, 131072):
                lib.plan(1, n, k, o)
                rows_now = min(rows, o[5])  # what a launch takes
                lib.plan(rows_now, n, k, o)
                bn, bm, tn, tm, splits, at_once, part, most, step, scratch, kb, waves, per, whole, launched = list(o)
                assert (tn - 1) * bn < n <= tn * bn and (tm - 1) * bm < rows_now <= tm * bm
                assert launched * 512 < 1 << 32 and launched == whole + (tn * tm - whole) * splits
                assert step % bm == 0 and at_once % step == 0 and at_once >= step
                assert at_once * kb * 256 <= scratch
                assert 1 <= splits <= min(kb, most) and most <= 64
                assert (splits - 1) * per < kb <= splits * per
                assert 0 <= whole <= tn * tm and whole % 256 == 0
                if splits > 1:
                    assert whole < tn * tm and (tn * tm - whole) * splits * bn * bm <= part
                own = lib.own(rows, n, kb)
                assert not own or bn == 16
                if bn == 16:  # the kernel without tiles: its LDS
                    assert splits == 1 and bm in (16, 32, 64) and waves in ((4, 8) if own else (8,))
                    assert not own or bm == 16
                    assert waves * bm // 16 * 1024 + own <= 160 * 1024


def test_oracle_rounds_to_the_nearest():
    """Against a search of all codes."""
    v = fm.VALUES[~np.isnan(fm.VALUES)]
    r = np.random.default_rng(1)
    x = np.concatenate([r.standard_normal(3000) * np.exp(3 * r.standard_normal(3000)), v, (v[1:] + v[:-1]) / 2])
    x = x[np.abs(x) <= 448]
    got = fm.rounded(x)
    best = np.abs(x[:, None] - v).min(1)
    assert np.all(np.abs(got - x) == best) and np.all(np.isin(got, v))
    w = (r.standard_normal((150, 160)) * np.exp(2 * r.standard_normal((150, 160)))).astype(np.float32)
    codes, scales = fm.quantized(w)
    for i in range(0, 150, 128):
        for j in range(0, 160, 128):
            part = w[i:i + 128, j:j + 128].astype(np.float64)
            s = float(scales[i // 128, j // 128])
            assert 224 < np.abs(part).max() / s <= 448 and np.log2(s) == np.rint(np.log2(s))
            assert np.array_equal(fm.VALUES[codes[i:i + 128, j:j + 128]], fm.rounded(part / s))
