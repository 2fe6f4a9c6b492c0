"""The paged 8-bit cache (qtts_paged_append_device, _attention_, _read_)
against its restatement in 64 bits (tests/paged_model.py).

Tolerances.  A rotated row is evaluated in 64 bits and rounded once: half an
f32 step, 2^-24 relative (and 2^-45 of the row's largest for the two 64-bit
evaluations).  Codes, scales and read values are then equal, bit for bit.
Attention: a score's rounding d is bounded by the sums that paged_model
returns (an f16 hi + lo query, 2^-22 of its largest; one f32 rounding for each
of the head_dim products), a probability's by 2 d, and an output's by that and
the f32 additions over the tokens, at most L/64 + 64 one after another, both
relative to sum p |v|."""
import numpy as np
import pytest
import torch

import paged_model as pm
import qtts

pytestmark = pytest.mark.gpu

ROPE_ROWS = 4096


def _rope(hd):
    freq = 1e6 ** (-np.arange(hd // 2) * 2 / hd)
    angle = np.arange(ROPE_ROWS)[:, None] * freq
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _ints(a):
    return _up(np.asarray(a, np.int32))


class Cache:
    """Device buffers of a cache; page tables in a shuffled pool."""

    def __init__(self, kv_heads, hd, page, slots, pages_each, seed=0, spare=2):
        self.kvh, self.hd, self.page, self.slots = kv_heads, hd, page, slots
        n = slots * pages_each + spare
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randperm(n, generator=g)[: slots * pages_each].int().view(slots, pages_each).cuda()
        # every byte starts as something that shows where it is read unwritten
        self.k_codes = torch.full((n, kv_heads, page, hd), 77, dtype=torch.int8, device="cuda")
        self.v_codes = torch.full((n, kv_heads, hd, page), 77, dtype=torch.int8, device="cuda")
        self.k_scales = torch.full((n, kv_heads), float("nan"), device="cuda")
        self.v_scales = torch.full((n, kv_heads), float("nan"), device="cuda")
        self.k_open = torch.full((slots, kv_heads, page, hd), float("nan"), device="cuda")
        self.v_open = torch.full((slots, kv_heads, page, hd), float("nan"), device="cuda")
        self.buffers = [self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.k_open, self.v_open]
        self.kv = qtts.PagedKv(*[b.data_ptr() for b in self.buffers], n, kv_heads, hd, page, slots)

    def seqs(self, starts, counts, rows=None, table=None, slots=None, max_rows=None):
        """A call over sequences at `starts` with `counts` rows each; the first
        len(starts) slots in order if none are named."""
        offsets = np.concatenate([[0], np.cumsum(counts)])
        slots = list(range(len(starts))) if slots is None else slots
        table = self.table[slots].contiguous() if table is None else table
        keep = [table, _ints(slots), _ints(starts), _ints(offsets)]
        s = qtts.PagedSeqs(len(starts), table.shape[1], int(offsets[-1]) if rows is None else rows,
                           max(counts) if max_rows is None else max_rows, *[t.data_ptr() for t in keep])
        s.keep = keep
        return s

    def append(self, ctx, seqs, k, v, **kw):
        torch.cuda.synchronize()
        ctx.paged_append_device(self.kv, seqs, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), **kw)
        ctx.synchronize()

    def attend(self, ctx, seqs, q, heads, window=0, out=None):
        out = torch.full((q.shape[0], heads * self.hd), 5.0, device="cuda") if out is None else out
        torch.cuda.synchronize()
        ctx.paged_attention_device(self.kv, seqs, heads, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0),
                                   scale=self.hd ** -0.5, window=window)
        ctx.synchronize()
        return out

    def read(self, ctx, seqs, lens=None):
        k, v = (torch.full((seqs.rows, self.kvh * self.hd), 9.0, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        ctx.paged_read_device(self.kv, seqs, 0 if lens is None else lens.data_ptr(), k.data_ptr(), k.stride(0),
                              v.data_ptr(), v.stride(0))
        ctx.synchronize()
        return k.cpu().numpy(), v.cpu().numpy()


def _normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("kvh,group,hd", [(2, 2, 128), (3, 1, 64), (1, 8, 128)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_and_read(ctx, page, kvh, group, hd, norm):
    """Ragged sequences, three calls each: new rows begin and end anywhere in a
    page; queries, cached values and everything behind them."""
    heads = kvh * group
    cos, sin = _rope(hd)
    dcos, dsin = _up(cos), _up(sin)
    qn, kn = ((1 + 0.1 * _normal(s, hd)).astype(np.float16) for s in (1, 2))
    dqn, dkn = _up(qn), _up(kn)
    c = Cache(kvh, hd, page, 4, 4)
    kw = dict(heads=heads, rope_cos=dcos.data_ptr(), rope_sin=dsin.data_ptr(), rope_rows=ROPE_ROWS)
    if norm:
        kw.update(q_norm=dqn.data_ptr(), k_norm=dkn.data_ptr(), eps=1e-6)
    qn, kn = (qn, kn) if norm else (None, None)
    starts = [0, 0, 0, 0]
    all_k, all_v = ([np.zeros((0, kvh, hd), np.float32) for _ in range(4)] for _ in range(2))
    for step, counts in enumerate([[1, page, page + 3, 0], [page - 1, 2 * page + 1, 1, page // 2], [3, 0, page, page]]):
        rows = sum(counts)
        width = (heads + 2 * kvh) * hd
        qkv = _normal(10 + step, rows + 2, width) * np.exp(0.5 * _normal(3, width))
        d = _up(qkv)
        q_out = torch.full((rows + 2, heads * hd + 4), 3.0, device="cuda")
        s = c.seqs(starts, counts)
        k, v = d[:, heads * hd:], d[:, (heads + kvh) * hd:]
        c.append(ctx, s, k, v, q=d.data_ptr(), ld_q=width, q_out=q_out.data_ptr(), ld_q_out=q_out.stride(0), **kw)
        got = q_out.cpu().numpy()
        assert np.all(got[rows:] == 3) and np.all(got[:, heads * hd:] == 3)
        at = 0
        for b, n in enumerate(counts):
            pos = starts[b] + np.arange(n)
            x = qkv[at:at + n].reshape(n, heads + 2 * kvh, hd)
            ref = pm.rotated(x[:, :heads], qn, 1e-6, cos, sin, pos)
            err = np.abs(got[at:at + n, :heads * hd].reshape(ref.shape) - ref)
            assert np.all(err <= 2.0 ** -24 * np.abs(ref) + 2.0 ** -45 * np.abs(ref).max(-1, keepdims=True))
            new_k = pm.rotated(x[:, heads:heads + kvh], kn, 1e-6, cos, sin, pos).astype(np.float32)
            all_k[b], all_v[b] = np.concatenate([all_k[b], new_k]), np.concatenate([all_v[b], x[:, heads + kvh:]])
            at += n
        starts = [a + n for a, n in zip(starts, counts)]
        lens = _ints(starts)
        k, v = c.read(ctx, c.seqs([0] * 4, starts), lens)
        at = 0
        for b, n in enumerate(starts):
            for rows_, held in ((k, pm.held(all_k[b], page)), (v, pm.held(all_v[b], page))):
                assert np.array_equal(rows_[at:at + n].reshape(n, kvh, hd), held), (step, b)
            at += n


def test_division_into_calls_does_not_matter(ctx):
    """The same tokens in one call, one by one and in odd parts: the same bytes."""
    page, hd, kvh, n = 32, 128, 2, 150
    k, v = _up(_normal(1, n, kvh * hd)), _up(_normal(2, n, kvh * hd))
    states = []
    for parts in ([n], [1] * n, [31, 1, 33, 64, 21], [100, 50]):
        c = Cache(kvh, hd, page, 1, 5)
        at = 0
        for m in parts:
            c.append(ctx, c.seqs([at], [m]), k[at:at + m], v[at:at + m])
            at += m
        used = c.table[0, : n // page].long()
        states.append([b[used].cpu() for b in c.buffers[:4]] + [b[0, :, : n % page].cpu() for b in c.buffers[4:]])
        rest = torch.ones(c.k_codes.shape[0], dtype=torch.bool, device="cuda")
        rest[used] = False
        assert torch.all(c.k_codes[rest] == 77) and torch.all(c.v_codes[rest] == 77)
    for other in states[1:]:
        for a, b in zip(states[0], other):
            assert torch.equal(a, b)


def test_going_back(ctx):
    """To a token of the open page, to its first, to a full page's first: the
    cache holds what was appended last, and attention sees no more."""
    kvh, hd, page = 2, 64, 32
    c = Cache(kvh, hd, page, 1, 5)
    k, v = np.zeros((0, kvh, hd), np.float32), np.zeros((0, kvh, hd), np.float32)
    for i, (start, rows) in enumerate([(0, 90), (70, 10), (64, 31), (32, 40), (72, 24), (96, 1), (96, 40), (0, 5)]):
        nk, nv, q = (_normal(s + 3 * i, rows, kvh * hd) for s in (1, 2, 3))
        c.append(ctx, c.seqs([start], [rows]), _up(nk), _up(nv))
        k, v = (np.concatenate([a[:start], b.reshape(rows, kvh, hd)]) for a, b in ((k, nk), (v, nv)))
        hk, hv = pm.held(k, page), pm.held(v, page)
        gk, gv = c.read(ctx, c.seqs([0], [start + rows]))
        assert np.array_equal(gk.reshape(hk.shape), hk) and np.array_equal(gv.reshape(hv.shape), hv)
        got = c.attend(ctx, c.seqs([start], [rows]), _up(q), kvh).cpu().numpy()
        _check(got.reshape(rows, kvh, hd), q.reshape(rows, kvh, hd), hk, hv, start, hd ** -0.5, 0)


def test_blocks_of_odd_values(ctx):
    """Zeros, subnormals, the largest floats, Inf and NaN, exact ties."""
    page, hd = 16, 64
    rows = []
    rows.append(np.zeros((page, hd), np.float32))
    rows.append(np.full((page, hd), 1e-42, np.float32) * np.arange(hd, dtype=np.float32))
    rows.append(_normal(1, page, hd) * np.float32(5e37))
    x = _normal(2, page, hd)
    x[3, 5] = np.inf
    rows.append(x)
    x = _normal(3, page, hd)
    x[15, 63] = np.nan
    rows.append(x)
    x = np.tile(np.arange(hd, dtype=np.float32) + 0.5, (page, 1))  # halves of 127 / 127 steps
    x[0, 0] = 127
    rows.append(x)
    x = -np.tile(np.arange(hd, dtype=np.float32) * 2 + 1, (page, 1))  # top 254: x / 2 is a tie
    x[7, 7] = 254
    rows.append(x)
    data = np.concatenate(rows)
    c = Cache(1, hd, page, 1, len(rows))
    d = _up(data)
    c.append(ctx, c.seqs([0], [len(data)]), d, d)
    ids = c.table[0].long()
    codes = c.k_codes[ids].cpu().numpy()[:, 0]
    vcodes = c.v_codes[ids].cpu().numpy()[:, 0].transpose(0, 2, 1)
    for i, x in enumerate(rows):
        ref, scale = pm.block(x)
        assert np.array_equal(codes[i], ref), i
        assert np.array_equal(vcodes[i], ref), i
        for s in (c.k_scales, c.v_scales):
            assert np.array_equal(s[ids].cpu().numpy()[i, 0], scale, equal_nan=True), i
    k, v = c.read(ctx, c.seqs([0], [len(data)]))
    held = pm.held(data[:, None], page)[:, 0]
    assert np.array_equal(k, held, equal_nan=True) and np.array_equal(v, held, equal_nan=True)


def _check(got, q, k, v, start, scale, window, absent=(), step=0.0):
    ref, mass, slack = pm.attention(q, k, v, start, scale, window, absent)
    err = np.abs(got - ref)
    tol = mass * (2 * slack[..., None] + (k.shape[0] / 64 + 64) * 2.0 ** -24)
    tol += step * np.abs(v).sum(0).repeat(q.shape[1] // v.shape[1], 0)
    assert np.all(np.isfinite(got))
    assert np.all(err <= tol), (float(err.max()), float((err / np.maximum(tol, 1e-30)).max()))
    # independent roundings add up as their squares do: far below the bound
    assert np.linalg.norm(err) <= 1e-5 * max(np.linalg.norm(ref), 1e-30)


def _filled(ctx, kvh, hd, page, starts, counts, seed=0, spread=1.0):
    """A cache with every sequence's tokens and what it holds, on the host."""
    ends = [a + n for a, n in zip(starts, counts)]
    c = Cache(kvh, hd, page, len(starts), -(-max(max(ends), 1) // page), seed)
    k, v = _normal(seed + 1, sum(ends), kvh * hd) * spread, _normal(seed + 2, sum(ends), kvh * hd)
    v *= np.exp(_normal(seed + 3, kvh * hd))
    dk, dv = _up(k), _up(v)
    if sum(ends):
        c.append(ctx, c.seqs([0] * len(ends), ends), dk, dv)
    held, at = [], 0
    for e in ends:
        held.append([pm.held(x[at:at + e].reshape(e, kvh, hd), page) for x in (k, v)])
        at += e
    return c, held


@pytest.mark.parametrize("kvh,group,hd", [(2, 2, 128), (2, 1, 64), (1, 5, 128), (1, 8, 64), (1, 16, 128), (1, 24, 64)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [0, 37])
def test_attention_single_tokens(ctx, page, kvh, group, hd, window):
    """One row per sequence at lengths from one to past several splits."""
    ends = [1, 2, page - 1, page, page + 1, 3 * page, 255, 256, 257, 1111]
    starts, counts = [e - 1 for e in ends], [1] * len(ends)
    c, held = _filled(ctx, kvh, hd, page, starts, counts, seed=page)
    q = _normal(5, len(ends), kvh * group * hd) * 2
    got = c.attend(ctx, c.seqs(starts, counts), _up(q), kvh * group, window).cpu().numpy()
    for b, (k, v) in enumerate(held):
        _check(got[b].reshape(1, -1, hd), q[b].reshape(1, -1, hd), k, v, starts[b], hd ** -0.5, window)


@pytest.mark.parametrize("kvh,group,hd", [(2, 2, 128), (2, 1, 64), (1, 6, 128)])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_attention_many_rows(ctx, page, kvh, group, hd, window):
    """Prompts and parts of prompts, ragged: rows of one sequence from none to
    several tiles, before and behind a page's border."""
    starts = [0, 0, 0, 7, page, 300, 5, 0]
    counts = [1, 0, page + 9, 2, 64, 65, 130, 3]
    c, held = _filled(ctx, kvh, hd, page, starts, counts, seed=page + 1)
    rows = sum(counts)
    q = _normal(6, rows + 3, kvh * group * hd) * 2
    out = c.attend(ctx, c.seqs(starts, counts, rows=rows + 3), _up(q), kvh * group, window).cpu().numpy()
    assert np.all(out[rows:] == 5.0)  # behind the last sequence: as it was
    at = 0
    for b, (k, v) in enumerate(held):
        n = counts[b]
        _check(out[at:at + n].reshape(n, kvh * group, hd), q[at:at + n].reshape(n, kvh * group, hd), k, v, starts[b],
               hd ** -0.5, window)
        at += n


@pytest.mark.parametrize("kvh,group,hd", [(1, 9, 64), (2, 16, 64), (1, 12, 128), (1, 3, 64), (3, 4, 128)])
@pytest.mark.parametrize("rows", [1, 2, 3])
def test_every_column_of_divided_tokens(ctx, kvh, group, hd, rows):
    """Groups that fill a tile, or the next one partly, with each sequence's
    tokens divided among blocks.

    Some columns here have one token with nearly all the probability and a code
    of 0 in a dimension, so that the output there is 1e-9 of V's size.  A weight
    is held to a least step, not to a share of itself: as an integer of which the
    column's largest is 2^27 or more (up to 4 columns), or as binary16 hi + lo,
    steps of 2^-24, of which the largest is 2^11 or more.  Half a step is 2^-28 or
    2^-36 of the largest weight, which is at most 1 of the sum, so an output is
    off by at most that times sum |v| beside what the others may be."""
    starts, counts = [2000, 700], [rows, rows]
    c, held = _filled(ctx, kvh, hd, 32, starts, counts, seed=12)
    q = _normal(13, 2 * rows, kvh * group * hd) * 2
    got = c.attend(ctx, c.seqs(starts, counts), _up(q), kvh * group).cpu().numpy()
    for b, (k, v) in enumerate(held):
        at = slice(b * rows, b * rows + rows)
        _check(got[at].reshape(rows, -1, hd), q[at].reshape(rows, -1, hd), k, v, starts[b], hd ** -0.5, 0,
               step=2.0 ** (-28 if rows * group <= 4 else -36))


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_long_cache(ctx, rows):
    """Past every split's length, with the scores of one far page on top."""
    kvh, hd, page, n = 1, 128, 64, 9000
    c, held = _filled(ctx, kvh, hd, page, [n], [rows], seed=3, spread=2.0)
    q = _normal(8, rows, 2 * hd) * 3
    got = c.attend(ctx, c.seqs([n], [rows]), _up(q), 2).cpu().numpy()
    _check(got.reshape(rows, 2, hd), q.reshape(rows, 2, hd), *held[0], n, hd ** -0.5, 0)


def test_strides_and_in_place(ctx):
    kvh, group, hd, page = 2, 2, 128, 32
    starts, counts = [40, 3], [1, 20]
    c, held = _filled(ctx, kvh, hd, page, starts, counts)
    q = _normal(4, 21, 3 * 4 * hd)
    d = _up(q)
    s = c.seqs(starts, counts)
    ref = c.attend(ctx, s, d[:, :4 * hd].contiguous(), 4)
    wide = torch.full((21, 5 * hd), 4.0, device="cuda")
    c.attend(ctx, s, d, 4, out=wide)
    assert torch.equal(wide[:, : 4 * hd], ref) and torch.all(wide[:, 4 * hd:] == 4)
    c.attend(ctx, s, d, 4, out=d)
    assert torch.equal(d[:, : 4 * hd], ref) and np.array_equal(d[:, 4 * hd:].cpu().numpy(), q[:, 4 * hd:])


@pytest.mark.parametrize("rows", [1, 33])
def test_absent_pages_and_sequences_left_out(ctx, rows):
    """Page ids outside the pool are left out; rows that see nothing, and
    sequences that cannot be served, are zeros, and nothing of theirs is written."""
    kvh, hd, page = 2, 64, 16
    n = 100
    starts, counts = [n - rows] * 6, [rows] * 6
    c, held = _filled(ctx, kvh, hd, page, starts, counts)
    table = c.table.clone()
    table[0, 0], table[0, 3] = -1, c.kv.num_pages
    table[1, :] = -2 ** 31
    slots = [0, 1, 6, 3, -1, 5]
    bad_starts = [n - rows, n - rows, n - rows, -1, n - rows, 7 * page - rows + 1]
    q = _normal(9, 6 * rows, kvh * hd)
    s = c.seqs(bad_starts, counts, table=table, slots=[0] * 6)
    s.keep.append(_ints(slots))
    s.slots = s.keep[-1].data_ptr()
    got = c.attend(ctx, s, _up(q), kvh).cpu().numpy().reshape(6, rows, kvh, hd)
    k, v = held[0]
    _check(got[0], q[:rows].reshape(rows, kvh, hd), k, v, n - rows, hd ** -0.5, 0,
           [t for t in range(n) if t // page in (0, 3)])
    k, v = held[1]
    _check(got[1], q[rows:2 * rows].reshape(rows, kvh, hd), k, v, n - rows, hd ** -0.5, 0, range(96))
    for b in range(2, 6):
        assert np.all(got[b] == 0), b
    before = [b.clone() for b in c.buffers]
    x = _up(_normal(10, 6 * rows, kvh * hd))
    q_out = torch.full((6 * rows, kvh * hd), 3.0, device="cuda")
    c.append(ctx, s, x, x, q=x.data_ptr(), ld_q=x.stride(0), heads=kvh, q_out=q_out.data_ptr(), ld_q_out=q_out.stride(0))
    assert torch.all(q_out.view(6, rows, -1)[2:] == 3) and torch.equal(q_out[: 2 * rows], x[: 2 * rows])
    for was, now in zip(before[4:], c.buffers[4:]):
        assert torch.equal(was[[2, 3, 4, 5]].nan_to_num(), now[[2, 3, 4, 5]].nan_to_num())
    own = table[0][(table[0] >= 0) & (table[0] < c.kv.num_pages)].long()
    rest = torch.ones(c.kv.num_pages, dtype=torch.bool, device="cuda")
    rest[own] = False
    for was, now in zip(before[:4], c.buffers[:4]):
        assert torch.equal(was[rest].nan_to_num(), now[rest].nan_to_num())
    k, v = c.read(ctx, s, _ints([n] * 6))
    assert np.all(k.reshape(6, rows, -1)[2:] == 0) and np.all(v.reshape(6, rows, -1)[2:] == 0)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_values_that_a_mask_hides(ctx, rows):
    """NaN and Inf in tokens that a row does not see leave it as it was: later
    open rows, tokens before the window, stale open rows, in K and in V."""
    kvh, hd, page, window = 2, 128, 64, 30
    start = 80
    n = start + rows
    c, held = _filled(ctx, kvh, hd, page, [start], [rows])
    q = _normal(9, rows, 2 * kvh * hd)
    s = c.seqs([start], [rows])
    ref = c.attend(ctx, s, _up(q), 2 * kvh, window)
    # the first page lies before the window of the last row, its scales too
    first = int(c.table[0, 0])
    if n - page >= window:
        for b in (c.k_scales, c.v_scales):
            b[first] = float("nan")
    if n // page == 1:  # tokens 64 ... n - 1 are open; n ... are stale
        for b, bad in ((c.k_open, float("inf")), (c.v_open, float("nan"))):
            b[0, :, n % page:] = bad
        low = max(0, n - rows - window + 1) - page  # open rows before the first row's window
        for b, bad in ((c.k_open, float("nan")), (c.v_open, float("-inf"))):
            b[0, :, : max(0, low)] = bad
    got = c.attend(ctx, s, _up(q), 2 * kvh, window)
    last = got[-1:] if n - page >= window else got
    assert torch.equal(last, ref[-1:] if n - page >= window else ref)
    # the last token, seen by the last row alone
    if rows > 1 and n // page == 1:
        c.v_open[0, :, (n - 1) % page, 3] = float("inf")
        c.k_open[0, 0, (n - 1) % page, 3] = float("nan")
        two = c.attend(ctx, s, _up(q), 2 * kvh, window)
        assert np.array_equal(two[:-1].cpu().numpy(), got[:-1].cpu().numpy(), equal_nan=True)
        assert torch.isnan(two[-1, : 2 * hd]).all()
        assert torch.isinf(two[-1, 2 * hd + 3]) and torch.isinf(two[-1, 3 * hd + 3])


@pytest.mark.parametrize("group,rows", [(1, 1), (4, 1), (6, 1), (2, 20)])
def test_many_small_weights_beside_a_large_one(ctx, group, rows):
    """One token with most of the probability and thousands that share the rest, in
    one block (of a batch that fills the card): roundings of small weights cancel,
    none is towards one side, which would show as some 2e-5 of the output here."""
    kvh, hd, page, n, pad = 1, 64, 64, 30000, 511
    c = Cache(kvh, hd, page, 1, -(-(n + rows) // page))
    q = np.tile(_normal(1, 1, hd), (rows, group)) + 0.01 * _normal(2, rows, group * hd)
    k, v = 0.02 * _normal(3, n + rows, hd), 0.5 + 0.5 * np.abs(_normal(4, n + rows, hd))
    k[1000] = q[0, :hd] * (np.log(4 * n) * hd ** 0.5 / (q[0, :hd] ** 2).sum())
    c.append(ctx, c.seqs([0], [n + rows]), _up(k), _up(v))
    s = c.seqs([0] * pad + [n], [0] * pad + [rows], table=c.table.expand(pad + 1, -1).contiguous(), slots=[0] * (pad + 1))
    got = c.attend(ctx, s, _up(q), group).cpu().numpy().reshape(rows, group, hd)
    hk, hv = (pm.held(x.reshape(n + rows, kvh, hd), page) for x in (k, v))
    ref, _, _ = pm.attention(q.reshape(rows, group, hd), hk, hv, n, hd ** -0.5, 0)
    assert np.abs(got / ref - 1).max() < 5e-6


SIZES = [0, 1e-44, 1e-42, 1e-39, 1e-37, 1e-30, 1, 1e30, 1e37, 3e38]


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("group,rows", [(1, 1), (6, 1), (1, 5), (8, 12), (2, 40)])
def test_values_of_every_size(ctx, group, rows, mixed):
    """V from zeros and the least floats to the largest, one size to a sequence or
    another in each page: pages whose values are nothing beside the others' keep
    their probabilities.

    Weights carry V's scale as its logarithm: it, its sum with a score and the
    difference from a reference are each rounded below 512, by 2^-16, and so is the
    reference: 4 ln 2 2^-16 < 2^-14 of a weight.  Then half a least step, 2^-28 of
    the largest weight (see above) for each token, times its block's largest value,
    and a step of the least floats."""
    kvh, hd, page, n, each = 1, 64, 16, 100, len(SIZES)
    k, q = _normal(1, each * n, kvh * hd), _normal(3, each * rows, kvh * group * hd)
    v = np.clip(_normal(2, each * n, kvh * hd), -1, 1)
    for b in range(each):
        for at in range(0, n, page):
            v[b * n + at:min(b * n + at + page, (b + 1) * n)] *= np.float32(SIZES[(b + mixed * at // page) % each])
    c = Cache(kvh, hd, page, each, 7)
    c.append(ctx, c.seqs([0] * each, [n] * each), _up(k), _up(v))
    got = c.attend(ctx, c.seqs([n - rows] * each, [rows] * each), _up(q), kvh * group).cpu().numpy()
    for b in range(each):
        hk, hv = (pm.held(x[b * n:(b + 1) * n].reshape(n, kvh, hd), page) for x in (k, v))
        mine = slice(b * rows, (b + 1) * rows)
        ref, mass, slack = pm.attention(q[mine].reshape(rows, -1, hd), hk, hv, n - rows, hd ** -0.5, 0)
        err = np.abs(got[mine].reshape(ref.shape) - ref)
        tol = mass * (2 * slack[..., None] + 2.0 ** -14 + (n / 64 + 64) * 2.0 ** -24)
        assert np.all(err <= tol + 2.0 ** -28 * n * np.abs(hv).max().astype(np.float64) + 2.0 ** -148), b


@pytest.mark.parametrize("group,rows", [(1, 4), (1, 12), (4, 12), (2, 40)])
def test_a_block_of_nan_in_the_middle_of_a_tile(ctx, group, rows):
    """A page that reads as NaN begins between two rows of one tile: those before
    it are as they were."""
    kvh, hd, page = 2, 128, 16
    start = 3 * page - rows // 2
    c, _ = _filled(ctx, kvh, hd, page, [start], [rows + page], seed=4)
    q, s = _up(_normal(5, rows + page, kvh * group * hd)), c.seqs([start], [rows + page])
    ref = c.attend(ctx, s, q, kvh * group)
    for scales in (c.v_scales, c.k_scales):
        kept = scales.clone()
        scales[int(c.table[0, 3])] = float("nan")
        got = c.attend(ctx, s, q, kvh * group)
        assert torch.equal(got[: rows // 2], ref[: rows // 2]) and torch.isnan(got[rows // 2:]).all()
        scales.copy_(kept)


def test_rows_of_nan_and_blocks_of_nan(ctx):
    """A NaN query gives its own row NaN; a block whose values read as NaN gives
    NaN to the rows that see it and to no others."""
    kvh, hd, page = 1, 64, 32
    starts, counts = [0], [100]
    c, held = _filled(ctx, kvh, hd, page, starts, counts)
    q = _normal(9, 100, hd)
    s = c.seqs(starts, counts)
    ref = c.attend(ctx, s, _up(q), 1)
    q[70, 5] = np.nan
    got = c.attend(ctx, s, _up(q), 1)
    keep = np.arange(100) != 70
    assert torch.isnan(got[70]).all() and torch.equal(got[keep], ref[keep])
    c.v_scales[int(c.table[0, 1])] = float("nan")
    got = c.attend(ctx, s, _up(q), 1)
    assert torch.equal(got[:32], ref[:32]) and torch.isnan(got[32:]).all()


def test_capture_and_replay(ctx):
    """A captured step follows what its arrays hold at each replay."""
    kvh, group, hd, page = 2, 2, 128, 16
    heads = kvh * group
    starts = _ints([30, 14])
    qkv = torch.zeros((2, (heads + 2 * kvh) * hd), device="cuda")
    q, out = torch.zeros((2, heads * hd), device="cuda"), torch.zeros((2, heads * hd), device="cuda")
    pool = Cache(kvh, hd, page, 2, 6, seed=5)
    x = _normal(1, 44, kvh * hd)
    d = _up(x)
    pool.append(ctx, pool.seqs([0, 0], [30, 14]), d, d)
    s = pool.seqs([30, 14], [1, 1])
    s.keep.append(starts)
    s.starts = starts.data_ptr()
    stream = torch.cuda.ExternalStream(ctx.stream)

    def step():
        at, ld = qkv.data_ptr(), qkv.stride(0)
        ctx.paged_append_device(pool.kv, s, at + 4 * heads * hd, ld, at + 4 * (heads + kvh) * hd, ld, heads=heads, q=at,
                                ld_q=ld, q_out=q.data_ptr(), ld_q_out=heads * hd)
        ctx.paged_attention_device(pool.kv, s, heads, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd,
                                   scale=hd ** -0.5)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    keys = [x[:30].reshape(30, kvh, hd), x[30:].reshape(14, kvh, hd)]
    vals = list(keys)
    for i in range(20):
        new = _normal(100 + i, 2, (heads + 2 * kvh) * hd)
        with torch.cuda.stream(stream):
            qkv.copy_(_up(new))
            starts.copy_(_ints([30 + i, 14 + i]))
            graph.replay()
        torch.cuda.synchronize()
        got = out.cpu().numpy().copy()
        new = new.reshape(2, -1, hd)
        for b in range(2):
            keys[b] = np.concatenate([keys[b], new[b:b + 1, heads:heads + kvh]])
            vals[b] = np.concatenate([vals[b], new[b:b + 1, heads + kvh:]])
            _check(got[b].reshape(1, heads, hd), new[b:b + 1, :heads], pm.held(keys[b], page), pm.held(vals[b], page),
                   len(keys[b]) - 1, hd ** -0.5, 0)
        again = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        step()
        ctx.synchronize()
        assert torch.equal(out, again)


def test_far_offsets(ctx):
    """A pool of more than 2^31 codes: pages at its end."""
    kvh, hd, page = 8, 128, 128
    per = kvh * hd * page
    pages = 2 ** 31 // per + 40
    c = Cache(kvh, hd, page, 1, 2, spare=0)
    c.k_codes = torch.zeros((pages, kvh, page, hd), dtype=torch.int8, device="cuda")
    c.v_codes = torch.zeros((pages, kvh, hd, page), dtype=torch.int8, device="cuda")
    c.k_scales, c.v_scales = (torch.zeros((pages, kvh), device="cuda") for _ in range(2))
    c.kv = qtts.PagedKv(*[b.data_ptr() for b in (c.k_codes, c.v_codes, c.k_scales, c.v_scales, c.k_open, c.v_open)],
                        pages, kvh, hd, page, 1)
    c.table = _ints([[pages - 1, pages - 3, 2]])
    n = 2 * page + 5
    k, v = _normal(1, n, kvh * hd), _normal(2, n, kvh * hd)
    c.append(ctx, c.seqs([0], [n]), _up(k), _up(v))
    gk, gv = c.read(ctx, c.seqs([0], [n]))
    hk, hv = pm.held(k.reshape(n, kvh, hd), page), pm.held(v.reshape(n, kvh, hd), page)
    assert np.array_equal(gk.reshape(hk.shape), hk) and np.array_equal(gv.reshape(hv.shape), hv)
    q = _normal(3, 1, kvh * hd)
    got = c.attend(ctx, c.seqs([n - 1], [1]), _up(q), kvh).cpu().numpy()
    _check(got.reshape(1, kvh, hd), q.reshape(1, kvh, hd), hk, hv, n - 1, hd ** -0.5, 0)


def test_refusals(ctx):
    c = Cache(2, 64, 16, 1, 2)
    x = torch.zeros((4, 128), device="cuda")
    s = c.seqs([0], [4])
    c.kv.page_size = 24
    for call in (lambda: c.append(ctx, s, x, x), lambda: c.attend(ctx, s, x, 2), lambda: c.read(ctx, s)):
        with pytest.raises(qtts.QttsError, match="page_size") as e:
            call()
        assert e.value.status == qtts.QTTS_ESHAPE
    c.kv.page_size = 16
    with pytest.raises(qtts.QttsError, match="heads"):
        c.attend(ctx, s, x, 3)
    with pytest.raises(qtts.QttsError, match="aligned"):
        ctx.paged_append_device(c.kv, s, x.data_ptr() + 4, 128, x.data_ptr(), 128)
    empty = c.seqs([0], [0], max_rows=0)
    c.append(ctx, empty, x, x)
    assert torch.all(c.k_codes == 77)
