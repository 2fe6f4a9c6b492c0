"""qtts_sample_rows_device on rows of which only some tokens are allowed (the
others -Inf), as a grammar or a range of a vocabulary leaves them: the token and
the share of the definition in 64 bits (test_gpu_sample_rows.definition).

The two sums differ by no more than 2^-45 of the largest weight for each kept
token (half a unit of 2^-44; less is left out): a draw differs from the
definition's only where the uniform number is nearer to a border than
2000 * 2^-45 = 6e-11, which a number of 24 bits is not but by an accident of the
seed, and a share by that and the half step of its rounding."""
import numpy as np
import pytest

import test_gpu_sample_rows as base

pytestmark = base.pytestmark

# on either side of the sizes where a row's maxima are of 4, 16 and 64 logits
VOCABS = [12288, 12289, 32768, 32769, 40000, 131072, 131073, 151936]


def allowed(how, n, vocab, r):
    if how == "adjacent":
        return int(r.integers(0, vocab - n + 1)) + np.arange(n)
    if how == "last":
        return vocab - n + np.arange(n)
    if how == "two places":  # within 64 logits each where there are few
        half = n // 2
        return np.concatenate([1000 + np.arange(half), vocab // 2 + np.arange(n - half)])
    return np.sort(r.choice(vocab, n, replace=False))


def masked(seed, vocab, n, rows, spread=2.0):
    r = np.random.default_rng(seed)
    x = np.full((rows, vocab), -np.inf, np.float32)
    for i, how in zip(range(rows), ["adjacent", "last", "two places", "scattered"] * rows):
        x[i, allowed(how, n, vocab, r)] = spread * r.standard_normal(n)
    return x, r.random(rows).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 10, 12, 64, 150, 640, 2000])
@pytest.mark.parametrize("vocab", VOCABS)
def test_few_allowed_tokens(ctx, vocab, n):
    """1 to 2000 allowed tokens, kept 2 to 3000, with and without top-p and min-p."""
    x, u = masked(vocab + n, vocab, n, 8)
    for k in (2, 20, 50, 200, 3000):
        base.check(ctx, x, u, [0.8] * 8, [k] * 8, ld=vocab + 1)
        base.check(ctx, x, u[::-1].copy(), [1.5] * 8, [k] * 8, [1.0, 0.9] * 4, [0.0, 0.0, 0.05, 0.05] * 2)


@pytest.mark.parametrize("vocab,n,k", [(40000, 3000, 1000), (131073, 9000, 400), (151936, 16000, 2000),
                                       (151936, 16000, 200), (524288, 100000, 3000), (131073, 122881, 2000)])
def test_many_allowed_tokens(ctx, vocab, n, k):
    """More than the kernels hold between them, fewer groups than top_k."""
    x, u = masked(n + k, vocab, n, 4)
    base.check(ctx, x, u, [0.9] * 4, [k] * 4)
    base.check(ctx, x, u[::-1].copy(), [2.0] * 4, [k] * 4, [0.95] * 4)


@pytest.mark.parametrize("top", [np.inf, 3e38])
def test_one_far_above(ctx, top):
    x, u = masked(5, 151936, 40, 4)
    x[np.arange(4), np.argmax(x, 1)] = top
    base.check(ctx, x, u, [0.8] * 4, [30] * 4)


@pytest.mark.parametrize("vocab,n,k", [(151936, 10, 50), (40000, 10, 50), (131072, 150, 20), (151936, 64, 50)])
def test_every_allowed_token_is_drawn(ctx, vocab, n, k):
    """A uniform number from the middle of each kept token's part of the sum."""
    x, _ = masked(n + vocab, vocab, n, 4, spread=1.0)
    for row in x:
        kept = base.definition(row, 0.9, k, 1.0, 0.0, 0.5)[2]
        kept = kept[row[kept] > -np.inf]  # fewer allowed than top_k: others follow, of no weight
        w = np.exp((row[kept].astype(np.float64) - row.max()) / 0.9)
        edges = np.concatenate([[0], np.cumsum(w) / w.sum()])
        u = (edges[:-1] + edges[1:]) / 2
        token, _ = base.draw(ctx, np.tile(row, (len(u), 1)), u, [0.9] * len(u), [k] * len(u))
        assert np.array_equal(token, kept)


@pytest.mark.parametrize("low", [np.finfo(np.float32).min, -1e4])
@pytest.mark.parametrize("vocab", [12288, 40000, 151936])
def test_masked_by_a_low_value(ctx, vocab, low):
    """A finite mask, which takes part in top-k and has no weight."""
    x, u = masked(vocab, vocab, 10, 4)
    y, v = masked(vocab + 1, vocab, vocab // 2, 4)
    for a, b in ((x, u), (y, v)):
        a = np.where(a == -np.inf, np.float32(low), a)
        base.check(ctx, a, b, [0.8] * 4, [50] * 4)
        base.check(ctx, a, b[::-1].copy(), [1.5] * 4, [0, 3, 2000, 0], [0.9, 1.0, 0.9, 1.0], [0.0, 0.0, 0.0, 0.05])
