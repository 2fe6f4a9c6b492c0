"""What an operation on a cache's pages writes beside the pool is an array of its own
(csrc/pages_plan.h, compiled for the host): refused where it is one of the pool's or
another of the call's, but for what a reservation lacks, which may take the place of
its starts or ends."""
import ctypes as C
import os
import subprocess

import pytest

import qtts
from conftest import PKG

GLUE = """
#include "pages_plan.h"
using namespace qtts;
extern "C" int remap(const qtts_paged_pool *p, const int32_t *s, const int32_t *t, const int32_t *c) {
    return check_remap(*p, s, t, 0, 0, c).status;
}
extern "C" int reserve(const qtts_paged_pool *p, const int32_t *s, const int32_t *e, const int32_t *l) {
    return check_reserve(*p, s, e, l).status;
}
extern "C" int compact(const qtts_paged_pool *p, const int32_t *f, const int32_t *t, const int32_t *l) {
    const Refusal r = check_compact(*p, f, t, l);
    return r.status == QTTS_OK ? check_compact_own(*p, f, t, l).status : r.status;
}
"""

OK, EINVAL = qtts.QTTS_OK, qtts.QTTS_EINVAL
NAMES = ("refs", "page_table", "slots", "source", "tokens", "starts", "ends", "from", "to", "live", "copied", "lacking")
AT = {n: (1 << 20) + 4096 * i for i, n in enumerate(NAMES)}


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("arrays")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    for f in (lib.remap, lib.reserve, lib.compact):
        f.argtypes = [C.c_void_p] * 4
    return lib


def _call(lib, name, args, **over):
    at = {**AT, **{k: AT.get(v) for k, v in over.items()}}
    pool = qtts.PagedPool(AT["refs"], AT["page_table"], AT["slots"], 100, 64, 5, 7)
    return getattr(lib, name)(C.byref(pool), *(at[a] for a in args))


REMAP, RESERVE, COMPACT = ("source", "tokens", "copied"), ("starts", "ends", "lacking"), ("from", "to", "live")


@pytest.mark.parametrize("name,args", [("remap", REMAP), ("reserve", RESERVE), ("compact", COMPACT)])
def test_arrays_of_their_own(lib, name, args):
    assert _call(lib, name, args) == OK
    assert _call(lib, name, args, **{args[2]: None}) == OK  # not wanted


@pytest.mark.parametrize("name,args,written,others", [
    ("remap", REMAP, "copied", ("refs", "page_table", "slots", "source", "tokens")),
    ("reserve", RESERVE, "lacking", ("refs", "page_table", "slots")),
    ("compact", COMPACT, "from", ("refs", "page_table", "slots", "to", "live")),
    ("compact", COMPACT, "to", ("refs", "page_table", "slots", "from", "live")),
    ("compact", COMPACT, "live", ("refs", "page_table", "slots", "from", "to")),
])
def test_refused(lib, name, args, written, others):
    for other in others:
        assert _call(lib, name, args, **{written: other}) == EINVAL, other


def test_lacking_in_place(lib):
    for other in ("starts", "ends"):
        assert _call(lib, "reserve", RESERVE, lacking=other) == OK
    assert _call(lib, "reserve", RESERVE, ends="starts") == OK
    assert _call(lib, "remap", REMAP, tokens="source") == OK
