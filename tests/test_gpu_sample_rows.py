"""qtts_sample_rows_device against its definition in 64 bits: the token has to
be the same one.  The operator's sums are exact to 2^-45 of the largest weight
and the definition's to 2^-53 a term, so that a draw could only differ where the
uniform number is nearer to a border than about 1e-11: the numbers drawn here
are not.  A share is a 64-bit quotient rounded once, over a sum good to 2^-45
for each token of the row."""
import numpy as np
import pytest
import torch

import qtts

pytestmark = pytest.mark.gpu


def definition(x, t, k, p, m, u):
    """(token, share, kept tokens) of one row of f32 logits."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any():
        return -1, np.nan, []
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, []
    if not t > 0:
        i = int(np.argmax(x))
        return i, 1.0, [i]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.where((x == -np.inf) | (top == np.inf), 0.0, np.exp((x - top) / t)))
    order = np.argsort(-x, kind="stable")
    if 0 < k < x.size:
        order = order[:k]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])])
        n = max(1, int((before[:-1] < max(p, 0.0) * before[-1]).sum()))
        order = order[:n]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = 0.0 if not u > 0 else min(u, 1.0)
    at = min(int((run <= u * run[-1]).sum()), int((run < run[-1]).sum()))
    return int(kept[at]), w[kept[at]] / run[-1], kept


def draw(ctx, x, u, t=None, k=None, p=None, m=None, ld=None):
    rows, vocab = x.shape
    ld = ld or vocab
    d = torch.full((rows, ld), 1e30, device="cuda")
    d[:, :vocab] = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
    args = {n: torch.from_numpy(np.asarray(a, ty)).cuda() for n, a, ty in (
        ("temperature", t, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32), ("min_p", m, np.float32))
        if a is not None}
    du = torch.from_numpy(np.asarray(u, np.float32)).cuda()
    token = torch.full((rows + 1,), 77, dtype=torch.int32, device="cuda")
    share = torch.full((rows + 1,), 77.0, device="cuda")
    torch.cuda.synchronize()
    ctx.sample_rows_device(d.data_ptr(), ld, rows, vocab, du.data_ptr(), token.data_ptr(), probs=share.data_ptr(),
                           **{n: a.data_ptr() for n, a in args.items()})
    ctx.synchronize()
    assert token[-1] == 77 and share[-1] == 77
    return token.cpu().numpy()[:-1], share.cpu().numpy()[:-1]


def check(ctx, x, u, t=None, k=None, p=None, m=None, ld=None):
    x = np.asarray(x, np.float32)
    rows, vocab = x.shape
    token, share = draw(ctx, x, u, t, k, p, m, ld)
    at = lambda a, i, off: off if a is None else float(np.float32(a[i]))
    for i in range(rows):
        ref, w, _ = definition(x[i], at(t, i, 1.0), int(at(k, i, 0)), at(p, i, 1.0), at(m, i, 0.0),
                               float(np.float32(u[i])))
        assert token[i] == ref, (i, token[i], ref)
        assert np.isnan(w) and np.isnan(share[i]) or abs(share[i] - w) <= w * (2.0 ** -24 + vocab * 2.0 ** -45 + 1e-12)


def rows_like_a_model(seed, rows, vocab):
    r = np.random.default_rng(seed)
    x = 2 * r.standard_normal((rows, vocab))
    for i in range(rows):
        at = r.integers(0, vocab, 30)
        x[i, at] = 8 + 2.5 * r.standard_normal(30)
        x[i, r.integers(0, vocab, vocab // 20)] = -np.inf
        x[i, r.integers(0, vocab)] = 9
    return x.astype(np.float32)


def settings(seed, rows):
    r = np.random.default_rng(seed)
    return dict(t=r.choice([0.0, 0.3, 0.8, 1.0, 1.7, 20.0], rows), k=r.choice([0, 1, 5, 50, 700, 10 ** 6], rows),
                p=r.choice([1.0, 0.99, 0.9, 0.5, 0.01], rows), m=r.choice([0.0, 0.0, 0.01, 0.2, 1.0], rows))


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 257, 1000, 2048, 4099, 16384, 16385, 32770, 50001, 151936, 524288])
def test_models_rows(ctx, vocab):
    rows = 24 if vocab < 100000 else 6
    u = np.random.default_rng(vocab).random(rows)
    check(ctx, rows_like_a_model(vocab, rows, vocab), u, **settings(vocab + 1, rows))


@pytest.mark.parametrize("name", ["t", "k", "p", "m", "none"])
@pytest.mark.parametrize("vocab", [777, 40000, 151936])
def test_one_setting_at_a_time(ctx, name, vocab):
    rows = 12
    s = settings(3, rows)
    u = np.random.default_rng(5).random(rows)
    check(ctx, rows_like_a_model(6, rows, vocab), u, **({name: s[name]} if name != "none" else {}), ld=vocab + 13)


@pytest.mark.parametrize("vocab", [300, 20000])
def test_every_kept_token_is_drawn_and_no_other(ctx, vocab):
    """A sweep of the uniform numbers finds each border."""
    x = rows_like_a_model(9, 1, vocab)[0]
    for t, k, p, m in ((0.9, 12, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (1.0, 0, 1.0, 0.15), (1.2, 20, 0.95, 0.02)):
        _, _, kept = definition(x, t, k, p, m, 0.5)
        w = np.exp((x[kept].astype(np.float64) - x.max()) / t)
        edges = np.concatenate([[0], np.cumsum(w) / w.sum()])
        u = np.concatenate([(edges[:-1] + edges[1:]) / 2, [0.0, 1.0 - 2.0 ** -24]])
        n = len(u)
        token, _ = draw(ctx, np.tile(x, (n, 1)), u, [t] * n, [k] * n, [p] * n, [m] * n)
        assert np.array_equal(token[:-2], kept) and token[-2] == kept[0] and token[-1] == kept[-1]


@pytest.mark.parametrize("vocab", [50, 3000, 30000, 151936])
def test_ties(ctx, vocab):
    """Equal logits go by index: a whole row of them, two levels, both zeros."""
    r = np.random.default_rng(vocab)
    x = np.zeros((9, vocab), np.float32)
    x[1] = -0.0
    x[2, r.integers(0, 2, vocab) == 1] = -0.0
    x[3] = r.integers(0, 2, vocab)
    x[4] = r.integers(-3, 3, vocab)
    x[5] = 1e-30
    x[6] = -3e38
    x[7, ::3] = 3e38
    x[8] = np.round(r.standard_normal(vocab) * 4) / 4
    for k, p, m in ((0, 1.0, 0.0), (7, 1.0, 0.0), (vocab - 1, 1.0, 0.0), (0, 0.5, 0.0), (0, 0.25, 1.0), (40, 0.7, 0.3)):
        u = r.random(9)
        check(ctx, x, u, [0.7] * 9, [k] * 9, [p] * 9, [m] * 9)
    check(ctx, x, r.random(9), [0.0] * 9)


@pytest.mark.parametrize("vocab", [5, 2000, 40000])
def test_odd_logits_and_settings(ctx, vocab):
    x = rows_like_a_model(4, 12, vocab)
    x[0, vocab // 2] = np.nan
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, vocab - 1] = -5
    x[3, :2] = np.inf
    x[4, :] = np.inf
    x[5, 1] = np.inf
    x[6] = np.linspace(-3e38, 3e38, vocab)
    x[7] = 1e-40 * np.arange(vocab)
    nan = float("nan")
    u = [0.3, 0.3, 0.3, 0.7, 0.999, 0.5, 0.5, 0.5, -1.0, 2.0, nan, 1.0]
    for t in (0.8, 0.0, nan, -2.0, 1e-30, 1e30, float("inf")):
        for p, m, k in ((1.0, 0.0, 0), (0.9, 0.05, 3), (nan, nan, -5), (0.0, 0.0, 0), (-1.0, 7.0, 4)):
            check(ctx, x, u, [t] * 12, [k] * 12, [p] * 12, [m] * 12)


def test_rows_do_not_go_by_their_neighbours(ctx):
    """One row alone, among others, twice: the same draw."""
    x = rows_like_a_model(8, 70, 5000)
    s, u = settings(9, 70), np.random.default_rng(1).random(70)
    token, share = draw(ctx, x, u, **s)
    again, share2 = draw(ctx, x, u, **s)
    assert np.array_equal(token, again) and np.array_equal(share, share2)
    for i in (0, 33, 69):
        one, _ = draw(ctx, x[i:i + 1], u[i:i + 1], **{n: a[i:i + 1] for n, a in s.items()})
        assert one[0] == token[i]


@pytest.mark.parametrize("vocab", [1500, 60000])
def test_capture_and_replay(ctx, vocab):
    rows = 5
    x = torch.zeros((rows, vocab), device="cuda")
    u, t = torch.zeros(rows, device="cuda"), torch.full((rows,), 0.9, device="cuda")
    k = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
    token = torch.zeros(rows, dtype=torch.int32, device="cuda")
    stream = torch.cuda.ExternalStream(ctx.stream)

    def step():
        ctx.sample_rows_device(x.data_ptr(), vocab, rows, vocab, u.data_ptr(), token.data_ptr(),
                               temperature=t.data_ptr(), top_k=k.data_ptr())

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i in range(4):
        lx, lu = rows_like_a_model(20 + i, rows, vocab), np.random.default_rng(i).random(rows).astype(np.float32)
        with torch.cuda.stream(stream):
            x.copy_(torch.from_numpy(lx))
            u.copy_(torch.from_numpy(lu))
            graph.replay()
        torch.cuda.synchronize()
        got = token.cpu().numpy().copy()
        for r in range(rows):
            assert got[r] == definition(lx[r], float(np.float32(0.9)), 40, 1.0, 0.0, float(lu[r]))[0]
        step()
        ctx.synchronize()
        assert np.array_equal(token.cpu().numpy(), got)


def test_refusals(ctx):
    x = torch.zeros((2, 8), device="cuda")
    for ld, vocab, status in ((7, 8, qtts.QTTS_ESHAPE), (8, 0, qtts.QTTS_ESHAPE), (1 << 20, 1 << 20, qtts.QTTS_ESHAPE)):
        with pytest.raises(qtts.QttsError) as e:
            ctx.sample_rows_device(x.data_ptr(), ld, 2, vocab, x.data_ptr(), x.data_ptr())
        assert e.value.status == status
    with pytest.raises(qtts.QttsError) as e:
        ctx.sample_rows_device(x.data_ptr(), 8, 2, 8, 0, x.data_ptr())
    assert e.value.status == qtts.QTTS_EINVAL
    ctx.sample_rows_device(0, 8, 0, 8, 0, 0)


@pytest.mark.parametrize("vocab", [8193, 12289, 70003])
def test_more_rows_than_the_scratch_holds(ctx, vocab):
    """Long rows share the context's scratch in turns: in each the draws that the
    same rows have among few."""
    x = np.tile(rows_like_a_model(31, 20, vocab), (20, 1))
    s, u = settings(32, 400), np.random.default_rng(33).random(400)
    token, share = draw(ctx, x, u, **s)
    for lo in range(0, 400, 50):
        t, p = draw(ctx, x[lo:lo + 50], u[lo:lo + 50], **{n: a[lo:lo + 50] for n, a in s.items()})
        assert np.array_equal(t, token[lo:lo + 50]) and np.array_equal(p, share[lo:lo + 50])
    check(ctx, x[::23], u[::23], **{n: a[::23] for n, a in s.items()})


@pytest.mark.parametrize("k", [64, 65, 257, 1999, 6000, 8300, 20000])
@pytest.mark.parametrize("vocab", [8200, 12288, 12289, 33000, 151936])
def test_many_candidates(ctx, k, vocab):
    """Few to more than are held between the kernels; with and without top-p after
    top-k, rows that do not begin on 16 bytes."""
    rows = 6
    r = np.random.default_rng(k)
    x = r.standard_normal((rows, vocab)).astype(np.float32)
    x[1] *= 6
    x[2, :vocab // 2] = -np.inf
    x[3, 100:4000] += 3  # most of them in one chunk
    x[4] = np.round(x[4] * 64) / 64
    p = [1.0, 0.9, 0.7, 0.95, 1.0, 0.3]
    check(ctx, x, r.random(rows), [0.7, 1.0, 1.3, 0.9, 2.0, 1.0], [k] * rows, p, [0.0, 0.0, 1e-3, 0.0, 0.01, 0.0], ld=vocab + 3)


@pytest.mark.parametrize("vocab", [8200, 12288, 12289, 33000, 151936])
def test_many_tokens_at_the_cut(ctx, vocab):
    """top-p alone, with from few to all of a row's tokens in one narrow step of
    weight, in one chunk or in all of them."""
    r = np.random.default_rng(vocab)
    x = np.full((5, vocab), -20.0, np.float32)
    for i, n in enumerate((300, 3000, 7000)):
        at = r.choice(min(vocab, 9000 if i % 2 else vocab), n, replace=False)
        x[i, at] = 1 + 1e-3 * r.standard_normal(n)
    x[3] = 1e-4 * r.standard_normal(vocab)
    x[4, 4096:8192] = 2 + 1e-4 * r.standard_normal(4096)
    for p in (0.9, 0.31):
        check(ctx, x, r.random(5), [1.0] * 5, None, [p] * 5, [0.0, 0.5, 0.0, 0.0, 0.9])
