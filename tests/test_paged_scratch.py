"""The paged attention's chunks' results in their scratch (csrc/paged_plan.h): the
kernel's own width of a column, for every number of pairs."""
import ctypes as C
import os
import subprocess

from conftest import PKG

GLUE = """
#include "paged_plan.h"
using namespace qtts;
static_assert(part_floats(64) >= 64 + 3 && part_floats(128) >= 128 + 3, "output, reference, sum and its power");
static_assert(part_floats(64) % 4 == 0 && part_floats(128) % 4 == 0, "rows on 16 bytes");
extern "C" void plan(long long pairs, long long cap, int columns, long long *o) {
    const AttnPlan p = attn_plan(pairs, cap, columns);
    o[0] = pairs - p.whole;
    o[1] = o[0] * p.nsplit * columns * part_floats(128);  // past the last float that is written
    o[2] = kPagedPartFloats; o[3] = kPagedCounters;
}
"""


def test_every_part_lies_in_the_scratch(tmp_path):
    (tmp_path / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(tmp_path / "glue.cpp"), "-o", str(tmp_path / "glue.so")], check=True)
    lib = C.CDLL(str(tmp_path / "glue.so"))
    out = (C.c_longlong * 4)()
    most = 0
    for pairs in list(range(1, 1100)) + [65536 * 3 + 7, 2 ** 24 - 1]:
        for cap in (16, 256, 257, 600, 2048, 32768, 1 << 30):
            for columns in (4, 16, 32):
                lib.plan(C.c_longlong(pairs), C.c_longlong(cap), columns, out)
                shared, floats, room, counters = list(out)
                assert shared <= counters
                if shared:
                    assert floats <= room
                    most = max(most, floats)
    assert most >= 512 * 32 * 132  # a full round of them was among these
