"""A limit of tokens that a sequence of the paged cache may reach
(qtts_paged_seqs.max_tokens), as the three calls keep it."""
import numpy as np
import pytest
import torch

import test_gpu_paged as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 7, 40])
def test_past_the_rotations_table(ctx, rows):
    """A sequence whose last token is one past the table beside one that ends with
    it, in the slots and pages of two that were there before: append leaves it out,
    and attention and read give zeros, not what the others had left."""
    kvh, group, hd, page, table = 2, 2, 64, 32, 75  # of 96 that the pages hold
    cos, sin = (base._up(a[:table]) for a in base._rope(hd))
    c = base.Cache(kvh, hd, page, 2, 3)
    old = base._up(base._normal(1, 192, kvh * hd))
    c.append(ctx, c.seqs([0, 0], [96, 96]), old, old)
    c.append(ctx, c.seqs([64, 64], [31, 31]), old[:62], old[:62])
    s = c.seqs([table - rows + 1, table - rows], [rows, rows])
    s.max_tokens = table
    x = base._up(base._normal(2, 2 * rows, kvh * group * hd))
    q = torch.full_like(x, 3.0)
    before = [b.clone() for b in c.buffers]
    c.append(ctx, s, x, x, heads=kvh * group, q=x.data_ptr(), ld_q=x.stride(0), q_out=q.data_ptr(),
             ld_q_out=q.stride(0), rope_cos=cos.data_ptr(), rope_sin=sin.data_ptr(), rope_rows=table)
    assert torch.all(q[:rows] == 3.0) and not torch.any(q[rows:] == 3.0)
    mine = c.table[0].long()
    for was, now in zip(before[:4], c.buffers[:4]):
        assert torch.equal(was[mine], now[mine])
    for was, now in zip(before[4:], c.buffers[4:]):
        was, now = was.nan_to_num(), now.nan_to_num()
        assert torch.equal(was[0], now[0]) and not torch.equal(was[1], now[1])
    out = c.attend(ctx, s, q, kvh * group)
    assert torch.all(out[:rows] == 0) and torch.isfinite(out[rows:]).all() and torch.all(out[rows:].abs().sum(1) > 0)
    for lens in (None, base._ints([table + 1, table])):
        k, v = c.read(ctx, s, lens)
        assert np.all(k[:rows] == 0) and np.all(v[:rows] == 0) and np.all(np.abs(k[rows:]).sum(1) > 0)
