"""The checks of the operations on a cache's pages (csrc/pages_plan.h), compiled
for the host: what a call refuses and with which status, and that whatever the
device arrays hold, what a kernel does with a row stays inside the call's
buffers; and which pages a row keeps, against a look at every token."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import qtts
from conftest import PKG

GLUE = """
#include "pages_plan.h"
using namespace qtts;
static const char *why;
static int told(const Refusal &r) { why = r.why; return r.status; }
extern "C" const char *reason() { return why ? why : ""; }
extern "C" int remap(const qtts_paged_pool *p, const int32_t *s, const int32_t *t, int w, int k, const int32_t *c) {
    return told(check_remap(*p, s, t, w, k, c));
}
extern "C" int reserve(const qtts_paged_pool *p, const int32_t *s, const int32_t *e, const int32_t *l) {
    return told(check_reserve(*p, s, e, l));
}
extern "C" int compact(const qtts_paged_pool *p, const int32_t *f, const int32_t *t, const int32_t *l) {
    return told(check_compact(*p, f, t, l));
}
extern "C" int pages(const qtts_paged_kv *a, const qtts_paged_kv *b, int n, const int32_t *f, const int32_t *t) {
    return told(check_copy_pages(*a, *b, n, f, t));
}
extern "C" int open_(const qtts_paged_kv *a, int n, const int32_t *f, const int32_t *t, const int32_t *k) {
    return told(check_copy_open(*a, n, f, t, k));
}
extern "C" int kept(int j, int tokens, int self, int page, int window, int sinks) {
    return page_kept(j, tokens, self, page, window, sinks);
}
extern "C" void heir(const qtts_paged_pool *p, const int32_t *s, const int32_t *t, int b, int *o) {
    const Heir h = heir_of(*p, s, t, b);
    o[0] = h.source; o[1] = h.tokens;
}
extern "C" void span(const qtts_paged_pool *p, int a, int e, int *o) {
    const Span s = reserve_span(*p, a, e);
    o[0] = s.first; o[1] = s.last;
}
"""

OK, EINVAL, ESHAPE, ERANGE = qtts.QTTS_OK, qtts.QTTS_EINVAL, qtts.QTTS_ESHAPE, qtts.QTTS_ERANGE
AT = 1 << 20  # an address that is never read


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("pages")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.reason.restype = C.c_char_p
    lib.remap.argtypes = [C.c_void_p] * 3 + [C.c_int, C.c_int, C.c_void_p]
    lib.reserve.argtypes = lib.compact.argtypes = [C.c_void_p] * 4
    lib.pages.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
    lib.open_.argtypes = [C.c_void_p, C.c_int] + [C.c_void_p] * 3
    return lib


def _pool(**over):
    v = dict(refs=AT, page_table=AT, slots=AT, num_pages=100, page_size=64, batch=5, max_pages=7)
    v.update(over)
    return qtts.PagedPool(*v.values())


@pytest.mark.parametrize("pool,status", [
    (dict(), OK), (dict(page_size=8), ESHAPE), (dict(page_size=48), ESHAPE), (dict(page_size=256), ESHAPE),
    (dict(num_pages=0), ESHAPE), (dict(num_pages=(1 << 22) - 64), OK), (dict(num_pages=(1 << 22) - 63), ERANGE),
    (dict(batch=-1), ESHAPE), (dict(batch=8192, max_pages=512), OK), (dict(batch=8193), ESHAPE),
    (dict(batch=8192, max_pages=513), ERANGE), (dict(max_pages=-1), ESHAPE),
    (dict(batch=1, max_pages=1 << 22), OK), (dict(batch=1, max_pages=1 << 23), ERANGE),
    (dict(batch=0, page_table=0, slots=0), OK), (dict(max_pages=0, page_table=0), OK), (dict(refs=0), EINVAL),
    (dict(refs=AT + 8), EINVAL), (dict(page_table=0), EINVAL), (dict(page_table=AT + 2), EINVAL),
    (dict(slots=0), EINVAL), (dict(slots=AT + 1), EINVAL), (dict(page_size=128, batch=0, max_pages=1 << 24), ERANGE),
])
def test_pools(lib, pool, status):
    p = C.byref(_pool(**pool))
    assert lib.remap(p, AT, AT, 0, 0, None) == status, lib.reason()
    assert lib.reserve(p, AT, AT, None) == status
    assert lib.compact(p, AT, AT + 4096, None) == status
    assert bool(lib.reason()) == (status != OK)


def test_arrays(lib):
    p = C.byref(_pool())
    assert lib.remap(p, None, AT, 5, 3, AT + 4096) == OK
    for args in ((AT, None, 0, 0, None), (AT + 2, AT, 0, 0, None), (AT, AT + 1, 0, 0, None), (AT, AT, 0, 0, AT + 2),
                 (AT, AT, -1, 0, None), (AT, AT, 0, -1, None)):
        assert lib.remap(p, *args) == EINVAL
    for args in ((None, AT, AT), (AT, None, AT), (AT + 2, AT, AT), (AT, AT + 2, AT), (AT, AT, AT + 2)):
        assert lib.reserve(p, *args) == EINVAL
    for args in ((None, AT, AT), (AT, None, AT), (AT + 2, AT, AT), (AT, AT + 2, AT), (AT + 4, AT, AT + 2), (AT, AT, None)):
        assert lib.compact(p, *args) == EINVAL
    assert lib.compact(C.byref(_pool(num_pages=1)), None, None, AT) == OK


def test_what_a_remap_writes_is_an_array_of_its_own(lib):
    names = ("source", "tokens", "slots", "page_table")
    for same in (None,) + names:
        at = {n: AT + 4096 * (i + 1) for i, n in enumerate(names)}
        p = C.byref(_pool(slots=at["slots"], page_table=at["page_table"]))
        copied = at[same] if same else AT + 4096 * 9
        assert lib.remap(p, at["source"], at["tokens"], 0, 0, copied) == (EINVAL if same else OK)


def _kv(**over):
    v = dict(k_codes=AT, v_codes=AT, k_scales=AT, v_scales=AT, k_open=0, v_open=0, num_pages=10, kv_heads=2,
             head_dim=128, page_size=64, num_slots=0)
    v.update(over)
    return qtts.PagedKv(*v.values())


@pytest.mark.parametrize("over,status", [
    (dict(), OK), (dict(head_dim=96), ESHAPE), (dict(page_size=24), ESHAPE), (dict(kv_heads=0), ESHAPE),
    (dict(kv_heads=1025), ESHAPE), (dict(num_pages=0), ESHAPE), (dict(num_pages=1 << 30), ERANGE),
    (dict(k_codes=0), EINVAL), (dict(v_codes=AT + 8), EINVAL), (dict(k_scales=0), EINVAL), (dict(v_scales=AT + 2), EINVAL),
])
def test_copied_pages(lib, over, status):
    a, good = _kv(**over), _kv(**{k: v for k, v in over.items() if k in ("head_dim", "page_size", "kv_heads")})
    assert lib.pages(C.byref(a), C.byref(good), 4, AT, AT) == status, lib.reason()
    assert lib.pages(C.byref(good), C.byref(a), 4, AT, AT) == status


def test_copied_pages_lists(lib):
    a = C.byref(_kv())
    assert lib.pages(a, C.byref(_kv(num_pages=999)), 4, AT, AT) == OK
    for over in (dict(head_dim=64), dict(page_size=32), dict(kv_heads=4)):
        assert lib.pages(a, C.byref(_kv(**over)), 4, AT, AT) == ESHAPE
    assert lib.pages(a, a, 0, None, None) == OK
    assert lib.pages(a, a, -1, AT, AT) == ESHAPE
    assert lib.pages(a, a, 1 << 23, AT, AT) == ERANGE
    assert lib.pages(a, a, 4, None, AT) == EINVAL and lib.pages(a, a, 4, AT, AT + 2) == EINVAL


def test_copied_slots(lib):
    kv = dict(k_codes=0, v_codes=0, k_scales=0, v_scales=0, k_open=AT, v_open=AT, num_slots=3, num_pages=0)
    a = C.byref(_kv(**kv))
    assert lib.open_(a, 4, AT, AT, AT) == OK and lib.open_(a, 0, None, None, None) == OK
    assert lib.open_(a, -1, AT, AT, AT) == ESHAPE and lib.open_(a, 1 << 22, AT, AT, AT) == ERANGE
    for args in ((None, AT, AT), (AT, None, AT), (AT, AT, None), (AT + 2, AT, AT), (AT, AT + 2, AT), (AT, AT, AT + 2)):
        assert lib.open_(a, 4, *args) == EINVAL
    for over, status in ((dict(num_slots=0), ESHAPE), (dict(k_open=0), EINVAL), (dict(v_open=AT + 8), EINVAL),
                         (dict(head_dim=32), ESHAPE), (dict(page_size=0), ESHAPE)):
        assert lib.open_(C.byref(_kv(**{**kv, **over})), 4, AT, AT, AT) == status


def test_pages_that_a_row_keeps(lib):
    r = np.random.default_rng(1)
    for _ in range(4000):
        page = int(r.choice([16, 32, 64, 128]))
        tokens, window, sinks = int(r.integers(0, 700)), int(r.choice([0, 1, 2, 16, 100, 129])), int(r.integers(0, 200))
        j, self = int(r.integers(0, 50)), int(r.integers(0, 2))
        there = j * page < tokens if self else (j + 1) * page <= tokens
        # any of its tokens seen by the next row, at position `tokens`
        seen = not window or any(t > tokens - window or t < sinks for t in range(j * page, (j + 1) * page))
        assert lib.kept(j, tokens, self, page, window, sinks) == (there and seen)
    big = 2 ** 31 - 1
    assert lib.kept(0, 1 << 30, 1, 16, big, 0) and lib.kept((1 << 26) - 1, 1 << 30, 1, 16, 2, 0)
    assert not lib.kept(0, 1 << 30, 1, 16, 1, 0) and lib.kept(0, 1 << 30, 1, 16, 1, big)


def test_any_device_arrays_stay_inside(lib):
    r = np.random.default_rng(2)
    edge = np.array([-2 ** 31, -1, 0, 1, 2, 3, 4, 5, 15, 16, 17, 447, 448, 449, 2 ** 30, 2 ** 31 - 1])
    out = (C.c_int * 2)()
    for _ in range(5000):
        source, tokens = (r.choice(edge, 5).astype(np.int32) for _ in range(2))
        p = _pool(max_pages=int(r.choice([0, 1, 7])))
        most = p.max_pages * 64
        for b in range(5):
            lib.heir(C.byref(p), C.c_void_p(source.ctypes.data), C.c_void_p(tokens.ctypes.data), b, out)
            assert -1 <= out[0] < 5 and 0 <= out[1] <= most
            assert out[0] == (source[b] if 0 <= source[b] < 5 else -1)
            for self in (0, 1):
                assert not lib.kept(p.max_pages, out[1], self, 64, 0, 0)
        a, e = (int(x) for x in r.choice(edge, 2))
        lib.span(C.byref(p), a, e, out)
        if a < 0 or e < 0 or e > most:
            assert (out[0], out[1]) == (-1, -1)
        else:
            assert 0 <= out[0] <= out[1] <= p.max_pages
            assert list(range(out[0], out[1])) == [j for j in range(p.max_pages) if j * 64 < e and (j + 1) * 64 > a]
