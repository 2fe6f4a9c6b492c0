"""A limit of tokens that a sequence of the paged cache may reach
(qtts_paged_seqs.max_tokens): the host's checks and the kernels' view of it
(csrc/paged_plan.h), compiled for the host."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import qtts
from conftest import PKG

GLUE = """
#include "paged_plan.h"
using namespace qtts;
extern "C" int attention(const qtts_paged_kv *kv, const qtts_paged_seqs *s, int heads, const float *q, int ld) {
    return check_attention(*kv, *s, heads, q, ld, 0.1f, 0, q, ld).status;
}
extern "C" long long cap(const qtts_paged_kv *kv, const qtts_paged_seqs *s) { return tokens_cap(*kv, *s); }
extern "C" int served(const qtts_paged_kv *kv, const qtts_paged_seqs *s) {
    return load_seq(*s, 0, kv->num_slots, tokens_cap(*kv, *s)).ok;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.cap.restype = C.c_longlong
    lib.attention.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int]
    return lib


AT = 1 << 20  # an address that is never read


def test_limits(lib):
    kv = qtts.PagedKv(AT, AT, AT, AT, AT, AT, 10, 2, 128, 64, 3)
    slots, offsets, starts = np.zeros(1, np.int32), np.array([0, 2], np.int32), np.zeros(1, np.int32)
    for most, cap in ((0, 256), (1, 1), (255, 255), (256, 256), (257, 256), (2 ** 31 - 1, 256)):
        s = qtts.PagedSeqs(1, 4, 2, 2, AT, slots.ctypes.data, starts.ctypes.data, offsets.ctypes.data, most)
        assert lib.cap(C.byref(kv), C.byref(s)) == cap
        assert lib.attention(C.byref(kv), C.byref(s), 4, AT, 512) == qtts.QTTS_OK
        for start in (0, cap - 3, cap - 2, cap - 1, cap, 2 ** 31 - 1):
            starts[0] = start
            assert lib.served(C.byref(kv), C.byref(s)) == (0 <= start <= cap - 2)
        starts[0] = 0
    s.max_tokens = -1
    assert lib.attention(C.byref(kv), C.byref(s), 4, AT, 512) == qtts.QTTS_ESHAPE
    # one that does not name it
    assert qtts.PagedSeqs(1, 4, 2, 2, AT, AT, AT, AT).max_tokens == 0
