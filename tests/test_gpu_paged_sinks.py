"""Attention over the paged cache with a window and first tokens that stay
visible (qtts_paged_attention_sinks_device), against 64 bits.  Tolerances are
those of tests/test_gpu_paged.py: a row sees other tokens, and is summed in the
same way.

Among many columns some have one token with nearly all the probability and a
code of 0 in a dimension, where the output is 1e-9 of V's size.  A weight is held
to a least step: as an integer of which the column's largest is 2^27 or more (up
to 4 columns), or as binary16 hi + lo, steps of 2^-24, of which the largest is
2^11 or more.  Half a step is 2^-28 or 2^-36 of the largest weight, which is at
most 1 of the sum, so an output is off by at most that times sum |v| over what it
sees, beside what the others may be."""
import numpy as np
import pytest
import torch

import qtts
import test_gpu_paged as paged

pytestmark = pytest.mark.gpu


def reference(q, k, v, start, scale, window, sinks, absent=()):
    """As paged_model.attention, with sinks."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    slack = np.zeros((rows, heads))
    token = np.arange(k.shape[0])
    gone = np.isin(token, np.asarray(list(absent), np.int64))
    for i in range(rows):
        seen = (token <= start + i) & ~gone & ((token > start + i - window) | (token < sinks))
        if not seen.any():
            continue
        for h in range(heads):
            kk, vv = k[seen, h // group].astype(np.float64), v[seen, h // group].astype(np.float64)
            x = q[i, h].astype(np.float64)
            s = kk @ x * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], mass[i, h] = w @ vv, w @ np.abs(vv)
            slack[i, h] = scale * (2.0 ** -22 * np.abs(x).max() * np.abs(kk).sum(1).max()
                                   + hd * 2.0 ** -24 * (np.abs(kk) @ np.abs(x)).max())
    return out, mass, slack


def _attend(ctx, c, s, q, heads, window, sinks):
    out = torch.full((q.shape[0], heads * c.hd), 5.0, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_attention_device(c.kv, s, heads, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0),
                               scale=c.hd ** -0.5, window=window, sinks=sinks)
    ctx.synchronize()
    return out


def _check(got, q, k, v, start, scale, window, sinks, absent=(), columns=None):
    """columns: of the call's longest sequence, where that is another one."""
    ref, mass, slack = reference(q, k, v, start, scale, window, sinks, absent)
    err = np.abs(got - ref)
    tol = mass * (2 * slack[..., None] + (k.shape[0] / 64 + 64) * 2.0 ** -24)
    group = q.shape[1] // v.shape[1]
    step = 2.0 ** (-28 if (columns or q.shape[0] * group) <= 4 else -36)
    tol += step * np.abs(v).sum(0).repeat(group, 0)
    assert np.all(np.isfinite(got))
    assert np.all(err <= tol), (float(err.max()), float((err / np.maximum(tol, 1e-30)).max()))
    assert np.linalg.norm(err) <= 1e-5 * max(np.linalg.norm(ref), 1e-30)


def _compare(ctx, kvh, group, hd, page, starts, counts, window, sinks, seed):
    c, held = paged._filled(ctx, kvh, hd, page, starts, counts, seed=seed)
    rows, heads = sum(counts), kvh * group
    q = paged._normal(6, rows + 2, heads * hd) * 2
    out = _attend(ctx, c, c.seqs(starts, counts, rows=rows + 2), paged._up(q), heads, window, sinks).cpu().numpy()
    assert np.all(out[rows:] == 5.0)
    at = 0
    for b, (k, v) in enumerate(held):
        n = counts[b]
        _check(out[at:at + n].reshape(n, heads, hd), q[at:at + n].reshape(n, heads, hd), k, v, starts[b], hd ** -0.5,
               window, sinks, columns=max(counts) * group)
        at += n


@pytest.mark.parametrize("window,sinks", [(1, 1), (1, 70), (37, 4), (37, 64), (37, 65), (200, 4), (200, 190), (64, 128),
                                          (500, 300), (2 ** 31 - 1, 5), (30, 2 ** 31 - 1)])
@pytest.mark.parametrize("kvh,group,hd", [(2, 2, 128), (2, 1, 64), (1, 8, 64), (1, 24, 128)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_single_tokens(ctx, page, kvh, group, hd, window, sinks):
    """At lengths around every border of page, step and sinks, to several splits."""
    ends = [1, 2, page, page + 1, 65, 127, 128, 129, 192, 193, 250, 257, 321, 1111]
    _compare(ctx, kvh, group, hd, page, [e - 1 for e in ends], [1] * len(ends), window, sinks, seed=page)


@pytest.mark.parametrize("window,sinks", [(1, 3), (50, 4), (20, 100), (130, 64), (300, 129)])
@pytest.mark.parametrize("kvh,group,hd", [(2, 2, 128), (2, 1, 64), (1, 6, 128)])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_many_rows(ctx, page, kvh, group, hd, window, sinks):
    starts = [0, 0, 0, 7, page, 300, 5, 700, 0]
    counts = [1, 0, page + 9, 2, 64, 65, 130, 40, 3]
    _compare(ctx, kvh, group, hd, page, starts, counts, window, sinks, seed=page + 1)


@pytest.mark.parametrize("kvh,group,hd,rows", [(8, 2, 64, 100), (16, 1, 64, 200), (8, 2, 128, 40), (64, 1, 128, 33)])
def test_tiles_of_32(ctx, kvh, group, hd, rows):
    """As many columns as the widest tiles are taken for."""
    starts, counts = [900, 200, 0, 411, 64, 130], [rows, rows - 1, rows, 17, rows - 5, rows]
    _compare(ctx, kvh, group, hd, 64, starts, counts, 90, 70, seed=5)


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("page", [32, 128])
def test_what_is_not_seen_is_not_read(ctx, page, rows):
    """The pages between sinks and window given back, in the table or still
    there and full of NaN; and pages of the sinks that are absent."""
    kvh, group, hd, window, sinks, n = 2, 2, 128, 150, 40, 2000
    c, held = paged._filled(ctx, kvh, hd, page, [n], [rows], seed=9)
    q = paged._up(paged._normal(7, rows, kvh * group * hd))
    s = c.seqs([n], [rows])
    first = _attend(ctx, c, s, q, kvh * group, window, sinks)
    _check(first.cpu().numpy().reshape(rows, -1, hd), q.cpu().numpy().reshape(rows, -1, hd), *held[0], n, hd ** -0.5,
           window, sinks)
    lost = torch.tensor([j for j in range(-(-(n + rows) // page)) if j * page >= sinks and (j + 1) * page <= n - window + 1],
                        device="cuda")
    assert len(lost) > 5
    ids = c.table[0][lost].long()
    c.k_scales[ids] = float("nan")
    c.v_scales[ids] = float("nan")
    c.k_codes[ids], c.v_codes[ids] = -128, -128
    assert torch.equal(_attend(ctx, c, s, q, kvh * group, window, sinks), first)
    c.table[0][lost] = -1
    s = c.seqs([n], [rows])
    assert torch.equal(_attend(ctx, c, s, q, kvh * group, window, sinks), first)
    c.table[0][0] = 2 ** 31 - 1
    s = c.seqs([n], [rows])
    got = _attend(ctx, c, s, q, kvh * group, window, sinks).cpu().numpy().reshape(rows, -1, hd)
    _check(got, q.cpu().numpy().reshape(rows, -1, hd), *held[0], n, hd ** -0.5, window, sinks, absent=range(page))


def test_without_sinks_or_window_as_before(ctx):
    """The same bits as attention without sinks."""
    kvh, group, hd, page = 2, 2, 64, 64
    starts, counts = [700, 40, 3000], [1, 70, 5]
    c, _ = paged._filled(ctx, kvh, hd, page, starts, counts, seed=2)
    q, s = paged._up(paged._normal(3, 76, kvh * group * hd)), c.seqs(starts, counts)
    out = [torch.zeros_like(q) for _ in range(2)]
    for window, sinks in ((0, 0), (0, 9), (100, 0)):
        for i, o in enumerate(out):
            args = (ctx.h, qtts.C.byref(c.kv), qtts.C.byref(s), kvh * group, q.data_ptr(), q.stride(0), hd ** -0.5, window)
            torch.cuda.synchronize()
            if i == 0:
                ctx.check(ctx.lib.qtts_paged_attention_device(*args, o.data_ptr(), o.stride(0)))
            else:
                ctx.check(ctx.lib.qtts_paged_attention_sinks_device(*args, sinks, o.data_ptr(), o.stride(0)))
            ctx.synchronize()
        assert torch.equal(*out)


@pytest.mark.parametrize("rows", [1, 12])
def test_odd_values(ctx, rows):
    """A query that is not finite makes its row NaN; an Inf among values that a
    row does not see does not reach it; a NaN sink reaches every row."""
    kvh, group, hd, page, window, sinks, n = 1, 2, 64, 32, 40, 3, 500
    c, held = paged._filled(ctx, kvh, hd, page, [n], [rows], seed=4)
    q = paged._normal(5, rows, group * hd)
    q[0, 5] = np.inf
    s = c.seqs([n], [rows])
    got = _attend(ctx, c, s, paged._up(q), group, window, sinks).cpu().numpy().reshape(rows, group, hd)
    assert np.all(np.isnan(got[0, 0])) and np.all(np.isfinite(got[0, 1]))
    q = paged._normal(5, rows, group * hd)
    c.v_scales[c.table[0][0].long()] = float("nan")
    got = _attend(ctx, c, s, paged._up(q), group, window, sinks).cpu().numpy()
    assert np.all(np.isnan(got))


def test_refusals(ctx):
    c, _ = paged._filled(ctx, 1, 64, 16, [5], [1])
    q, s = torch.zeros((1, 64), device="cuda"), c.seqs([5], [1])
    torch.cuda.synchronize()
    for bad in (dict(sinks=-1, window=4), dict(sinks=-2 ** 31), dict(sinks=3, window=-1)):
        with pytest.raises(qtts.QttsError) as e:
            ctx.paged_attention_device(c.kv, s, 1, q.data_ptr(), 64, q.data_ptr(), 64, scale=1.0, **bad)
        assert e.value.status == qtts.QTTS_EINVAL
