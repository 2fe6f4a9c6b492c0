"""Which kernel each shape of tests/fp8_shapes.py goes to (csrc/fp8_plan.h, compiled
for the host): a plan that sends one elsewhere fails here, not by leaving a kernel
without a test."""
import ctypes as C
import os
import subprocess

import pytest

import fp8_shapes as fs
from conftest import PKG

GLUE = """
#include "fp8_plan.h"
using namespace qtts;
extern "C" void plan(int rows, int n, int k, long long *o) {
    const Fp8Plan p = fp8_plan(rows, n, k);
    o[0] = p.bn; o[1] = p.bm; o[2] = p.splits; o[3] = p.whole;
    o[4] = fp8_own_rows(rows, n, fp8_blocks(k)); o[5] = rows <= fp8_rows_at_once(k);
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("shapes")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    return C.CDLL(str(d / "glue.so"))


@pytest.mark.parametrize("shape,kernel", [*fs.TILES.items(), *fs.DEEP.items(), *fs.FEW.items()])
def test_kernel(lib, shape, kernel):
    o = (C.c_longlong * 6)()
    lib.plan(*shape, o)
    side, rows_a_block, splits, whole, own, at_once = list(o)
    assert at_once
    if side == 16:
        assert kernel == (16, "own" if own else rows_a_block)
    else:
        assert not own and kernel == (side, fs.WHOLE if splits == 1 else fs.PARTLY if whole else fs.DIVIDED)


def test_every_kernel_has_a_shape():
    assert {(s, d) for s in (64, 128, 256) for d in (fs.WHOLE, fs.DIVIDED, fs.PARTLY)} - set(fs.TILES.values()) == {
        (256, fs.DIVIDED)}  # which no plan takes: fewer tiles of 128 cost less
