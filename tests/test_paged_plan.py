"""The paged cache's and the row sampler's checks (csrc/paged_plan.h), compiled
for the host: what a call refuses and with which status, and that whatever the
device arrays of a call hold, a sequence as the kernels read it stays inside
the call's buffers."""
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
static const char *why;
static int told(const Refusal &r) { why = r.why; return r.status; }
extern "C" const char *reason() { return why ? why : ""; }
extern "C" int append(const qtts_paged_kv *kv, const qtts_paged_seqs *s, const qtts_paged_rows *r) {
    return told(check_append(*kv, *s, *r));
}
extern "C" int attention(const qtts_paged_kv *kv, const qtts_paged_seqs *s, int heads, const float *q, int ld_q,
                         float scale, int window, const float *out, int ld_out) {
    return told(check_attention(*kv, *s, heads, q, ld_q, scale, window, out, ld_out));
}
extern "C" int read_(const qtts_paged_kv *kv, const qtts_paged_seqs *s, const int32_t *lens, const float *k, int ld_k,
                     const float *v, int ld_v) {
    return told(check_read(*kv, *s, lens, k, ld_k, v, ld_v));
}
extern "C" int sample(const float *l, int64_t ld, int rows, int vocab, const qtts_row_sampler *p, const float *u,
                      const int32_t *t, const float *pr) {
    return told(check_sample_rows(l, ld, rows, vocab, *p, u, t, pr));
}
extern "C" void plan(long long pairs, long long cap, int columns, long long *o) {
    const AttnPlan p = attn_plan(pairs, cap, columns);
    o[0] = p.whole; o[1] = p.nsplit; o[2] = kPagedMaxSplits; o[3] = kPagedPartFloats; o[4] = kPagedCounters;
}
extern "C" void shape(const qtts_paged_kv *kv, const qtts_paged_seqs *s, int heads, long long *o) {
    const AttnShape a = attn_shape(*kv, *s, heads);
    o[0] = a.mode; o[1] = a.tiles; o[2] = a.whole; o[3] = a.blocks;
}
extern "C" int chunk(int span, int nsplit, int round) { return chunk_of(span, nsplit, round); }
extern "C" void seq(const qtts_paged_seqs *s, int b, int slots, long long cap, int *o) {
    const PagedSeq q = load_seq(*s, b, slots, cap);
    o[0] = q.start; o[1] = q.rows; o[2] = q.row0; o[3] = q.slot; o[4] = q.ok;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "glue.cpp").write_text(GLUE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG, "csrc"), str(d / "glue.cpp"), "-o", str(d / "glue.so")], check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.reason.restype = C.c_char_p
    lib.attention.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_float, C.c_int, C.c_void_p,
                              C.c_int]
    lib.read_.argtypes = [C.c_void_p] * 4 + [C.c_int, C.c_void_p, C.c_int]
    lib.sample.argtypes = [C.c_void_p, C.c_int64, C.c_int, C.c_int] + [C.c_void_p] * 4
    lib.seq.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_longlong, C.c_void_p]
    return lib


AT = 1 << 20  # an address that is never read


def _kv(**over):
    v = dict(k_codes=AT, v_codes=AT, k_scales=AT, v_scales=AT, k_open=AT, v_open=AT, num_pages=10, kv_heads=2,
             head_dim=128, page_size=64, num_slots=3)
    v.update(over)
    return qtts.PagedKv(*v.values())


def _seqs(**over):
    v = dict(batch=2, max_pages=4, rows=5, max_rows=3, page_table=AT, slots=AT, starts=AT, row_offsets=AT)
    v.update(over)
    return qtts.PagedSeqs(*v.values())


def _rows(**over):
    v = dict(q=AT, k=AT, v=AT, q_out=AT, heads=4, ld_q=512, ld_k=256, ld_v=256, ld_q_out=512, q_norm=AT, k_norm=AT,
             eps=1e-6, rope_rows=100, rope_cos=AT, rope_sin=AT)
    v.update(over)
    return qtts.PagedRows(*v.values())


OK, EINVAL, ESHAPE, ERANGE = qtts.QTTS_OK, qtts.QTTS_EINVAL, qtts.QTTS_ESHAPE, qtts.QTTS_ERANGE

CACHE_AND_SEQS = [
    (dict(), dict(), OK),
    (dict(head_dim=64), dict(), OK),
    (dict(head_dim=96), dict(), ESHAPE),
    (dict(head_dim=256), dict(), ESHAPE),
    (dict(page_size=16), dict(), OK),
    (dict(page_size=8), dict(), ESHAPE),
    (dict(page_size=48), dict(), ESHAPE),
    (dict(page_size=256), dict(), ESHAPE),
    (dict(num_pages=0), dict(), ESHAPE),
    (dict(num_pages=1 << 30), dict(), ERANGE),
    (dict(num_pages=(1 << 30) - 1), dict(), OK),
    (dict(num_pages=-1), dict(), ESHAPE),
    (dict(kv_heads=0), dict(), ESHAPE),
    (dict(num_slots=0), dict(), ESHAPE),
    (dict(k_codes=0), dict(), EINVAL),
    (dict(v_codes=AT + 8), dict(), EINVAL),
    (dict(k_scales=AT + 2), dict(), EINVAL),
    (dict(v_scales=0), dict(), EINVAL),
    (dict(k_open=AT + 4), dict(), EINVAL),
    (dict(v_open=0), dict(), EINVAL),
    (dict(), dict(batch=-1), ESHAPE),
    (dict(), dict(batch=65537), ESHAPE),
    (dict(), dict(batch=0, slots=0), OK),
    (dict(), dict(rows=0, max_rows=0, starts=0), OK),
    (dict(), dict(rows=-1), ESHAPE),
    (dict(), dict(max_rows=-1), ESHAPE),
    (dict(), dict(max_rows=6), ESHAPE),
    (dict(), dict(max_pages=-1), ESHAPE),
    (dict(), dict(max_pages=(1 << 24) + 1), ERANGE),
    (dict(), dict(page_table=0), EINVAL),
    (dict(), dict(max_pages=0, page_table=0), OK),
    (dict(), dict(slots=0), EINVAL),
    (dict(), dict(starts=0), EINVAL),
    (dict(), dict(row_offsets=0), EINVAL),
    (dict(), dict(row_offsets=AT + 2), EINVAL),
    (dict(), dict(rows=(1 << 30) + 1), ERANGE),
]


@pytest.mark.parametrize("kv,seqs,status", CACHE_AND_SEQS)
def test_cache_and_sequences(lib, kv, seqs, status):
    k, s = _kv(**kv), _seqs(**seqs)
    wide = k.head_dim * 4
    assert lib.append(C.byref(k), C.byref(s), C.byref(_rows(ld_q=wide, ld_q_out=wide))) == status, lib.reason()
    assert lib.attention(C.byref(k), C.byref(s), 4, AT, wide, 0.1, 0, AT, wide) == status
    assert lib.read_(C.byref(k), C.byref(s), None, AT, wide, AT, wide) == status
    assert bool(lib.reason()) == (status != OK)


@pytest.mark.parametrize("rows,status", [
    (dict(q=0, q_out=0, heads=0, q_norm=0), OK), (dict(q_norm=0), EINVAL), (dict(k_norm=0), EINVAL),
    (dict(q_norm=0, k_norm=0, eps=-1.0), OK), (dict(eps=-1e-6), EINVAL), (dict(eps=float("nan")), EINVAL),
    (dict(rope_cos=0), EINVAL), (dict(rope_sin=0), EINVAL), (dict(rope_cos=0, rope_sin=0, rope_rows=0), OK),
    (dict(rope_rows=0), EINVAL), (dict(rope_cos=AT + 4), EINVAL), (dict(q_norm=AT + 2), EINVAL),
    (dict(heads=3), ESHAPE), (dict(heads=0), ESHAPE), (dict(heads=1026), ESHAPE), (dict(q_out=0), EINVAL),
    (dict(k=0), EINVAL), (dict(v=0), EINVAL), (dict(k=AT + 4), EINVAL), (dict(ld_k=255), EINVAL),
    (dict(ld_k=252), ESHAPE), (dict(ld_v=1024), OK), (dict(ld_q=508), ESHAPE), (dict(ld_q=1024), EINVAL),
    (dict(ld_q=1024, q_out=AT + 4096), OK), (dict(ld_q_out=510), EINVAL),
])
def test_append_rows(lib, rows, status):
    assert lib.append(C.byref(_kv()), C.byref(_seqs()), C.byref(_rows(**rows))) == status, lib.reason()


@pytest.mark.parametrize("args,status", [
    ((4, AT, 512, 0.1, 0, AT, 512), OK), ((4, AT, 512, 0.1, 7, AT + 512, 1024), OK),
    ((5, AT, 640, 0.1, 0, AT, 640), ESHAPE), ((4, None, 512, 0.1, 0, AT, 512), EINVAL),
    ((4, AT, 512, 0.1, 0, None, 512), EINVAL), ((4, AT, 512, 0.1, -1, AT, 512), EINVAL),
    ((4, AT, 512, float("inf"), 0, AT, 512), EINVAL), ((4, AT, 508, 0.1, 0, AT, 512), ESHAPE),
    ((4, AT, 512, 0.1, 0, AT, 1024), EINVAL), ((4, AT + 4, 512, 0.1, 0, AT, 512), EINVAL),
])
def test_attention_arguments(lib, args, status):
    assert lib.attention(C.byref(_kv()), C.byref(_seqs()), *args) == status, lib.reason()


def test_read_arguments(lib):
    kv, s = C.byref(_kv()), C.byref(_seqs())
    assert lib.read_(kv, s, AT, AT, 256, None, 0) == OK
    assert lib.read_(kv, s, AT, None, 0, AT, 256) == OK
    assert lib.read_(kv, s, AT + 1, AT, 256, AT, 256) == EINVAL
    assert lib.read_(kv, s, AT, AT, 252, AT, 256) == ESHAPE
    assert lib.read_(kv, s, AT, AT, 256, AT + 4, 256) == EINVAL


@pytest.mark.parametrize("args,status", [
    ((AT, 100, 3, 100), OK), ((AT, 99, 3, 100), ESHAPE), ((AT, 1 << 40, 3, 1 << 19), OK),
    ((AT, 1 << 40, 3, (1 << 19) + 1), ESHAPE), ((AT, 100, 3, 0), ESHAPE), ((AT, 100, -1, 100), ESHAPE),
    ((None, 100, 0, 100), OK), ((None, 100, 3, 100), EINVAL), ((AT + 2, 100, 3, 100), EINVAL),
])
def test_sample_arguments(lib, args, status):
    p = qtts.RowSampler(0, 0, 0, 0)
    assert lib.sample(*args, C.byref(p), AT, AT, None) == status, lib.reason()
    if status == OK and args[2]:
        assert lib.sample(*args, C.byref(p), None, AT, None) == EINVAL
        assert lib.sample(*args, C.byref(p), AT, None, None) == EINVAL
        for i in range(4):
            p = qtts.RowSampler(*[AT + (2 if j == i else 0) for j in range(4)])
            assert lib.sample(*args, C.byref(p), AT, AT, None) == EINVAL


def test_any_device_arrays_stay_inside(lib):
    r = np.random.default_rng(7)
    edge = np.array([-2 ** 31, -2 ** 31 + 1, -1, 0, 1, 2, 3, 5, 63, 64, 255, 256, 257, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1])
    out = np.zeros(5, np.int32)
    served = 0
    for _ in range(20000):
        offsets = r.choice(edge, 3).astype(np.int32)
        starts, slots = (r.choice(edge, 2).astype(np.int32) for _ in range(2))
        rows = int(r.choice([1, 4, 300]))
        most, cap, num_slots = int(r.integers(1, rows + 1)), int(r.choice([0, 16, 256, 1 << 30])), int(r.choice([1, 3]))
        s = _seqs(rows=rows, max_rows=most, starts=starts.ctypes.data, slots=slots.ctypes.data,
                  row_offsets=offsets.ctypes.data)
        for b in range(2):
            lib.seq(C.byref(s), b, num_slots, cap, out.ctypes.data)
            start, n, row0, slot, ok = (int(v) for v in out)
            assert 0 <= row0 and 0 <= n <= most and row0 + n <= rows
            first, last = int(offsets[b]), int(offsets[b + 1])
            if 0 <= first <= last <= rows and last - first <= most:
                assert (row0, n) == (first, last - first)
            if ok:
                assert 0 <= start and start + n <= cap and 0 <= slot < num_slots
                served += n > 0
    assert served > 100


def test_attention_plans(lib):
    """Every pair gets its blocks, a round's scratch and counters hold the
    shared ones, and the chunks of any span cover it."""
    out = (C.c_longlong * 5)()
    for pairs in list(range(1, 1600)) + [4096, 5000, 65536 * 3 + 7]:
        for cap, columns in ((16, 4), (256, 32), (257, 4), (2048, 32), (32768, 16), (1 << 30, 32)):
            lib.plan(C.c_longlong(pairs), C.c_longlong(cap), columns, out)
            whole, nsplit, most, part, counters = list(out)
            assert 0 <= whole <= pairs and nsplit >= 1
            shared = pairs - whole
            if shared == 0:
                continue
            assert nsplit > 1 and shared <= counters and nsplit <= most and nsplit <= -(-cap // 256)
            assert shared * nsplit * 32 * 130 <= part
            assert shared * nsplit <= 3 * 512 // 2 and whole % 512 == 0
    for span in list(range(1, 700)) + [32761, 100000]:
        for nsplit in (1, 2, 3, 16, 256):
            for step in (256, 512):
                chunk = lib.chunk(span, nsplit, step)
                assert chunk % step == 0 and chunk * nsplit >= span and chunk < span / nsplit + step + 1


@pytest.mark.parametrize("append,attention,read,kv,seqs", [
    (OK, OK, OK, dict(), dict(rows=1 << 20, max_rows=1 << 20)),
    (OK, OK, OK, dict(kv_heads=4), dict(batch=65536, rows=65536, max_rows=1)),
    (ERANGE, ERANGE, ERANGE, dict(kv_heads=256), dict(batch=65536, rows=65536, max_rows=1)),
    (ERANGE, ERANGE, OK, dict(kv_heads=4), dict(batch=65536, rows=1 << 20, max_rows=1 << 10)),
    (ERANGE, ERANGE, ERANGE, dict(), dict(batch=2, rows=1 << 30, max_rows=1 << 30)),
])
def test_more_blocks_than_a_launch_holds(lib, append, attention, read, kv, seqs):
    """2^24 blocks of 256 threads: refused before anything is enqueued."""
    k, s = _kv(**kv), _seqs(**seqs)
    heads = 2 * k.kv_heads
    wide = heads * k.head_dim
    got = lib.append(C.byref(k), C.byref(s), C.byref(_rows(heads=heads, ld_q=wide, ld_q_out=wide, ld_k=wide, ld_v=wide)))
    assert got == append, lib.reason()
    assert lib.attention(C.byref(k), C.byref(s), heads, AT, wide, 0.1, 0, AT, wide) == attention, lib.reason()
    assert lib.read_(C.byref(k), C.byref(s), None, AT, wide, AT, wide) == read, lib.reason()


def test_columns_of_a_tile(lib):
    """Few columns on int8 products, tiles of 32 only where they fill most of a
    round; always enough tiles for all columns."""
    out = (C.c_longlong * 4)()
    for batch, kvh, group, rows, mode in ((1, 8, 2, 1, 0), (64, 8, 4, 1, 0), (64, 8, 5, 1, 1), (4, 8, 2, 8, 1),
                                          (64, 8, 16, 1, 1), (64, 8, 17, 1, 2), (1, 8, 2, 512, 1), (1, 8, 2, 768, 2),
                                          (16, 8, 2, 32, 1), (16, 8, 2, 33, 2)):
        k, s = _kv(kv_heads=kvh), _seqs(batch=batch, rows=batch * rows, max_rows=rows)
        lib.shape(C.byref(k), C.byref(s), kvh * group, out)
        got, tiles, whole, blocks = list(out)
        each = (4, 16, 32)[got]
        assert got == mode and (tiles - 1) * each < group * rows <= tiles * each
        assert batch * kvh * tiles <= blocks and whole <= batch * kvh * tiles
