"""The paged cache's attention in tiles of 32 columns, which it takes where a
batch has several hundred of them: the cases of test_gpu_paged.py with empty
sequences in front of their own, as a padded batch has them.  `pairs` tiles (of
a kv head each): 400 of a block each; of 530 the last ones, which are the real
sequences' first rows, are divided among blocks."""
import pytest
import torch

import paged_model as pm
import test_gpu_paged as base

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[400, 530])
def padded(request, monkeypatch):
    """Sets a Cache's calls up with that many pairs, for `group` query heads to a
    kv head."""
    plain = base.Cache.seqs

    def start(group):
        def seqs(self, starts, counts, rows=None, table=None, slots=None, max_rows=None):
            each = self.kvh * -(-max(counts) * group // 32)
            pad = max(0, -(-request.param // each) - len(starts))
            slots = list(range(len(starts))) if slots is None else list(slots)
            table = self.table[slots] if table is None else table
            table = torch.cat([table[:1].expand(pad, -1), table]).contiguous()
            return plain(self, [0] * pad + list(starts), [0] * pad + list(counts), rows, table, [0] * pad + slots,
                         max_rows)
        monkeypatch.setattr(base.Cache, "seqs", seqs)
    return start


@pytest.mark.parametrize("kvh,group,hd", [(2, 2, 128), (2, 1, 64), (1, 6, 128), (1, 16, 64)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_many_rows(ctx, padded, page, kvh, group, hd, window):
    padded(group)
    base.test_attention_many_rows(ctx, page, kvh, group, hd, window)


@pytest.mark.parametrize("rows", [9, 40, 200])
def test_long_cache(ctx, padded, rows):
    padded(2)
    base.test_long_cache(ctx, rows)


def test_strides_and_in_place(ctx, padded):
    padded(2)
    base.test_strides_and_in_place(ctx)


@pytest.mark.parametrize("rows", [9, 40])
def test_values_that_a_mask_hides(ctx, padded, rows):
    padded(2)
    base.test_values_that_a_mask_hides(ctx, rows)


def test_rows_of_nan_and_blocks_of_nan(ctx, padded):
    padded(1)
    base.test_rows_of_nan_and_blocks_of_nan(ctx)


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("group,rows", [(1, 40), (8, 12)])
def test_values_of_every_size(ctx, padded, group, rows, mixed):
    padded(group)
    base.test_values_of_every_size(ctx, group, rows, mixed)


@pytest.mark.parametrize("group,rows", [(2, 40), (4, 12)])
def test_a_block_of_nan_in_the_middle_of_a_tile(ctx, padded, group, rows):
    padded(group)
    base.test_a_block_of_nan_in_the_middle_of_a_tile(ctx, group, rows)


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64)])
def test_absent_pages(ctx, padded, hd, page):
    """Pages outside the pool, in tiles of 32 columns; a sequence without any."""
    padded(1)
    kvh, rows, n = 2, 40, 3 * page + 40
    c, held = base._filled(ctx, kvh, hd, page, [n - rows] * 3, [rows] * 3)
    c.table[0, 0], c.table[0, 2] = -1, c.kv.num_pages
    c.table[1, :] = -2 ** 31
    q = base._normal(9, 3 * rows, kvh * hd)
    got = c.attend(ctx, c.seqs([n - rows] * 3, [rows] * 3), base._up(q), kvh).cpu().numpy().reshape(3, rows, kvh, hd)
    q = q.reshape(3, rows, kvh, hd)
    full = n // page * page
    for b, absent in ((0, [t for t in range(full) if t // page in (0, 2)]), (1, range(full)), (2, ())):
        base._check(got[b], q[b], *held[b], n - rows, hd ** -0.5, 0, absent)
