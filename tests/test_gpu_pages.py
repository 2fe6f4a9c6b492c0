"""The operations on a paged cache's pages (qtts_paged_remap_device, _reserve_,
_compact_, _copy_pages_, _copy_open_) against their restatement with lists
(tests/pages_model.py).  All results are whole numbers or copies: equal."""
import numpy as np
import pytest
import torch

import pages_model as model
import qtts

pytestmark = pytest.mark.gpu


def _up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _ints(a):
    return _up(np.asarray(a, np.int32))


class Pool:
    """A table whose rows share pages, hold none in places, and a pool with
    pages that the caller keeps for himself."""

    def __init__(self, seed, batch, wide, pages, page, fill=0.6):
        r = np.random.default_rng(seed)
        self.page, self.pages = page, pages
        table = np.full((batch, wide), -1, np.int64)
        own = r.permutation(pages)[:int(pages * fill)]
        at = 0
        for b in range(batch):
            n = int(r.integers(0, wide + 1))
            keep = int(r.integers(0, n + 1)) if b and r.random() < 0.4 else 0
            table[b, :keep] = table[b - 1, :keep]
            k = min(n - keep, len(own) - at)
            table[b, keep:keep + k] = own[at:at + k]
            at += k
        gone = r.random(table.shape)
        table[gone < 0.05] = -1
        table[gone > 0.98] = pages + 3  # outside the pool: no page
        refs = np.bincount(table[(table >= 0) & (table < pages)], minlength=pages)
        refs[r.permutation(pages)[:pages // 20]] += 1
        refs[(refs == 0) & (r.random(pages) < 0.1)] = -2  # free as well
        self.host = (table.tolist(), refs.tolist(), (r.permutation(batch) + 5).tolist())
        self.d_table, self.d_refs, self.d_slots = _ints(table), _ints(refs), _ints(self.host[2])
        self.pool = qtts.PagedPool(self.d_refs.data_ptr(), self.d_table.data_ptr(), self.d_slots.data_ptr(), pages,
                                   page, batch, wide)

    def now(self):
        return self.d_table.tolist(), self.d_refs.tolist(), self.d_slots.tolist()


SHAPES = [(1, 1, 1, 16), (1, 40, 50, 64), (5, 7, 60, 128), (64, 127, 7000, 64), (64, 128, 9000, 16), (65, 128, 400, 32),
          (1100, 5, 3000, 16), (1500, 9, 20000, 32), (8192, 3, 12000, 64), (3, 9000, 40000, 16), (2, 0, 10, 16)]


def _turn(seed, p):
    """Sources and lengths, some of them nonsense."""
    r = np.random.default_rng(seed)
    batch, wide = p.pool.batch, p.pool.max_pages
    source = np.where(r.random(batch) < 0.5, np.arange(batch), r.integers(0, batch, batch))
    source[r.random(batch) < 0.2] = -1
    odd = r.random(batch)
    source[odd < 0.02] = batch + 7
    source[odd > 0.98] = -2 ** 31
    tokens = r.integers(0, wide * p.page + 1, batch)
    tokens[r.random(batch) < 0.3] //= p.page
    tokens = np.where(r.random(batch) < 0.2, tokens // p.page * p.page, tokens)
    odd = r.random(batch)
    tokens[odd < 0.02] = -5
    tokens[odd > 0.98] = 2 ** 31 - 1
    return source.tolist(), tokens.tolist()


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 0), (300, 70), (16, 16), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_remap(ctx, shape, window, sinks):
    p = Pool(sum(shape), *shape)
    for turn in range(3):  # the second and third on what the one before left
        before = p.now()
        source, tokens = _turn(7 * turn + window % 1000, p)
        ds, dt, copied = _ints(source), _ints(tokens), torch.full((p.pool.batch + 1,), 99, device="cuda").int()
        torch.cuda.synchronize()
        ctx.paged_remap_device(p.pool, 0 if turn == 1 else ds.data_ptr(), dt.data_ptr(), window=window, sinks=sinks,
                               copied=copied.data_ptr())
        ctx.synchronize()
        *ref, ref_copied = model.remap(*before, None if turn == 1 else source, tokens, p.page, window, sinks)
        assert list(p.now()) == ref
        assert copied.tolist() == ref_copied + [99]
        assert sorted(p.now()[2]) == sorted(before[2])


@pytest.mark.parametrize("fill", [0.1, 0.6, 0.95])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_reserve(ctx, shape, fill):
    p = Pool(sum(shape) + 1, *shape, fill=fill)
    r = np.random.default_rng(3)
    batch, most = p.pool.batch, p.pool.max_pages * p.page
    for turn in range(3):
        before = p.now()
        starts = r.integers(0, most + 1, batch)
        ends = np.minimum(starts + np.where(r.random(batch) < 0.7, 1, r.integers(0, most + 1, batch)), most)
        odd = r.random(batch)
        starts[odd < 0.03], ends[odd > 0.97] = -1, most + 1
        ends[(odd > 0.4) & (odd < 0.45)] = 0
        starts[(odd > 0.45) & (odd < 0.47)] = 2 ** 31 - 1
        ends[(odd > 0.47) & (odd < 0.48)] = -2 ** 31
        ds, de, lacking = _ints(starts), _ints(ends), torch.full((batch + 1,), 99, device="cuda").int()
        torch.cuda.synchronize()
        ctx.paged_reserve_device(p.pool, ds.data_ptr(), de.data_ptr(), 0 if turn == 2 else lacking.data_ptr())
        ctx.synchronize()
        table, refs, ref_lacking = model.reserve(*before[:2], starts.tolist(), ends.tolist(), p.page)
        assert list(p.now()) == [table, refs, before[2]]
        assert lacking.tolist() == ([99] * batch if turn == 2 else ref_lacking) + [99]


@pytest.mark.parametrize("fill", [0.0, 0.3, 0.7, 1.0])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_compact(ctx, shape, fill):
    p = Pool(sum(shape) + 2, *shape, fill=fill)
    before, most = p.now(), p.pages // 2
    moves, live = torch.full((2, most + 1), 99, device="cuda").int(), _ints([0])
    torch.cuda.synchronize()
    ctx.paged_compact_device(p.pool, moves[0].data_ptr(), moves[1].data_ptr(), live.data_ptr())
    ctx.synchronize()
    table, refs, frm, to, n = model.compact(*before[:2])
    assert list(p.now()) == [table, refs, before[2]]
    assert moves.tolist() == [frm + [99], to + [99]] and live.tolist() == [n]
    ctx.paged_compact_device(p.pool, moves[0].data_ptr(), moves[1].data_ptr(), 0)  # packed already
    ctx.synchronize()
    assert list(p.now()) == [table, refs, before[2]] and moves[:, :most].flatten().tolist() == [-1] * (2 * most)


def _cache(seed, pages, kvh, page, hd, slots=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-128, 128, (2, pages, kvh, page * hd), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.randn((2, pages, kvh), generator=g, device="cuda")
    opened = torch.randn((2, slots, kvh, page, hd), generator=g, device="cuda")
    kv = qtts.PagedKv(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(),
                      opened[0].data_ptr(), opened[1].data_ptr(), pages, kvh, hd, page, slots)
    return kv, codes, scales, opened


@pytest.mark.parametrize("kvh,page,hd", [(8, 64, 128), (1, 16, 64), (3, 128, 64), (5, 32, 128), (300, 16, 64)])
def test_copy_pages(ctx, kvh, page, hd):
    """Within a cache and to another one; pairs outside either pool are left out."""
    for other in (False, True):
        a, ca, sa, _ = _cache(1, 40, kvh, page, hd)
        b, cb, sb, _ = _cache(2, 23, kvh, page, hd) if other else (a, ca, sa, None)
        a.k_open = a.v_open = 0
        frm = [3, 39, -1, 40, 2 ** 31 - 1, 5, 30, 3, 31]
        to = [0, 22, 1, 2, 4, -2 ** 31, 40, 7, 9]
        rc, rs = cb.clone(), sb.clone()
        for x, y in zip(frm, to):
            if 0 <= x < 40 and 0 <= y < b.num_pages:
                rc[:, y], rs[:, y] = ca[:, x], sa[:, x]
        df, dt = _ints(frm), _ints(to)
        torch.cuda.synchronize()
        ctx.paged_copy_pages_device(a, b, len(frm), df.data_ptr(), dt.data_ptr())
        ctx.synchronize()
        assert torch.equal(cb, rc) and torch.equal(sb, rs)
        ctx.paged_copy_pages_device(a, b, 0, 0, 0)


@pytest.mark.parametrize("kvh,page,hd", [(8, 64, 128), (1, 16, 64), (3, 128, 64), (5, 32, 128)])
def test_copy_open(ctx, kvh, page, hd):
    kv, _, _, opened = _cache(3, 1, kvh, page, hd, slots=40)
    kv.k_codes = kv.v_codes = kv.k_scales = kv.v_scales = 0
    frm = [0, 0, 1, -1, 2, 40, 3, 4, 5, 6, 7, 7]
    to = [20, 21, 22, 23, 40, 24, -7, 4, 25, 26, 27, 28]
    tokens = [1, page, page + 1, 5, 5, 5, 5, 5, -1, 2 * page - 1, 0, 2 ** 31 - 1]
    ref = opened.clone()
    for x, y, t in zip(frm, to, tokens):
        if 0 <= x < 40 and 0 <= y < 40 and t >= 0:
            ref[:, y, :, :t % page] = opened[:, x, :, :t % page]
    df, dt, dn = _ints(frm), _ints(to), _ints(tokens)
    torch.cuda.synchronize()
    ctx.paged_copy_open_device(kv, len(frm), df.data_ptr(), dt.data_ptr(), dn.data_ptr())
    ctx.synchronize()
    assert torch.equal(opened, ref)
    ctx.paged_copy_open_device(kv, 0, 0, 0, 0)


def test_no_rows(ctx):
    """A pool without sequences is packed all the same."""
    refs = _ints([0, 1, 0, 2, 0])
    pool = qtts.PagedPool(refs.data_ptr(), 0, 0, 5, 16, 0, 0)
    moves, live = _ints([[9, 9], [9, 9]]), _ints([9])
    torch.cuda.synchronize()
    ctx.paged_remap_device(pool, 0, 0)
    ctx.paged_reserve_device(pool, 0, 0)
    ctx.paged_compact_device(pool, moves[0].data_ptr(), moves[1].data_ptr(), live.data_ptr())
    ctx.synchronize()
    assert refs.tolist() == [2, 1, 0, 0, 0] and moves.tolist() == [[3, -1], [0, -1]] and live.tolist() == [2]


@pytest.mark.parametrize("wide", [100, 300])  # in one block, and through scratch
def test_graph(ctx, wide):
    """A step's calls captured and replayed on other lengths, with plain calls
    that use the same scratch between."""
    p, q = Pool(1, 30, wide, 5000, 16, fill=0.4), Pool(2, 40, 400, 9000, 16)
    r = np.random.default_rng(5)
    most = wide * 16
    ds, dt, de = _ints([0] * 30), _ints([0] * 30), _ints([0] * 30)
    copied, lacking = _ints([0] * 30), _ints([0] * 30)
    moves, live = torch.zeros((2, 2500), device="cuda").int(), _ints([0])

    def call():
        ctx.paged_remap_device(p.pool, ds.data_ptr(), dt.data_ptr(), window=200, sinks=20, copied=copied.data_ptr())
        ctx.paged_reserve_device(p.pool, dt.data_ptr(), de.data_ptr(), lacking.data_ptr())
        ctx.paged_compact_device(p.pool, moves[0].data_ptr(), moves[1].data_ptr(), live.data_ptr())

    stream = torch.cuda.ExternalStream(ctx.stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
    other = _ints(r.integers(0, 6400, 40))
    for turn in range(5):
        state = p.now()
        source, _ = _turn(turn, p)
        tokens = r.integers(0, most + 1, 30)
        ends = np.minimum(tokens + r.integers(1, 100, 30), most)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            ds.copy_(_ints(source)), dt.copy_(_ints(tokens)), de.copy_(_ints(ends))
            ctx.paged_remap_device(q.pool, 0, other.data_ptr())
            g.replay()
            ctx.paged_remap_device(q.pool, 0, other.data_ptr())
        torch.cuda.synchronize()
        table, refs, slots, c = model.remap(*state, source, tokens.tolist(), 16, 200, 20)
        table, refs, short = model.reserve(table, refs, tokens.tolist(), ends.tolist(), 16)
        table, refs, frm, to, n = model.compact(table, refs)
        assert p.now() == (table, refs, slots) and copied.tolist() == c and lacking.tolist() == short
        assert moves.tolist() == [frm, to] and live.tolist() == [n]
