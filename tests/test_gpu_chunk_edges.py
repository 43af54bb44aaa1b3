"""Chunk attention at its borders: every key once, scores of any size, infinities and NaN of values whose weight is nothing."""
import numpy as np
import pytest

import paged_step_util as ps

pytestmark = pytest.mark.gpu

HEADS = [(4, 2, 128), (8, 1, 64), (3, 1, 64), (2, 2, 256), (16, 8, 128)]
# decode, drafts, tiles of few and of many rows, over caches that are cut into pieces and that are not
BATCHES = [([1], [9001]), ([1, 1, 2], [9000, 3, 4095]), ([16], [8999]), ([40, 1], [9000, 4608]), ([70], [9057]), ([300], [5000]),
           ([1] * 20, list(range(120, 140))), ([4] * 9, [4090 + 11 * i for i in range(9)]), ([129, 7], [0, 640]), ([1], [0]), ([65], [127])]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", range(len(BATCHES)))
def test_every_visible_key_counts_once(dtype, heads, batch):
    n, start = BATCHES[batch]
    q, k, v, table = ps.picking(n, start, *heads, dtype, seed=batch)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, max(n), max(s + m for s, m in zip(start, n)))
    assert ps.picking_error(got, *ps.picking_want(q, k, v, table, n, start)) <= 0.25


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [1, 16, 70])
def test_long_cache_to_the_bound_of_the_weights_that_are_held(dtype, n):
    """as the long-cache test of every type, with nothing lost above 2^-35 of a row's largest weight"""
    rng = np.random.default_rng(n)
    ns, start = [n, 1], [9000, 3]
    table, n_pages = ps.pages_for(ns, start, rng)
    q = (3 * rng.standard_normal((n + 1, 4, 128))).astype(dtype)
    k, v = (rng.standard_normal((n_pages, 2, 128, 128)).astype(dtype) for _ in range(2))
    got = ps.chunk(q, k, v, table, ps.cu_of(ns), start, n, 9000 + n)
    want, tol = ps.chunk_want(q, k, v, table, ns, start, 9000 + n, lost=2.0 ** -35)
    ps.assert_within(got, want, tol)


def largest_wins(n, start, hq, hk, d, dtype, top, down):
    """Scores so far apart that the largest take all: queries +-top, keys top / 4, top / 2 or top (down: negated) in all places.
    The result is the mean of the values of the keys with a row's largest score; its error: sums of equal terms in fp32 and
    one rounding."""
    rng = np.random.default_rng(d)
    table, n_pages = ps.pages_for(n, start, rng)
    q = np.full((sum(n), hq, d), top, dtype)
    k = np.broadcast_to((-1 if down else 1) * top * rng.choice([0.25, 0.5, 1], (n_pages, hk, 128, 1), p=[0.55, 0.42, 0.03]),
                        (n_pages, hk, 128, d)).astype(dtype)
    v = rng.standard_normal((n_pages, hk, 128, d)).astype(dtype)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, max(n), max(s + m for s, m in zip(start, n)))
    cu, g = ps.cu_of(n), hq // hk
    for b in range(len(n)):
        pages = table[b, :(start[b] + n[b] + 127) // 128]
        for h in range(hk):
            K, V = (p[pages, h].reshape(-1, d).astype(np.float64) for p in (k, v))
            for i in range(n[b]):
                m = start[b] + i + 1
                at = np.nonzero(K[:m, 0] == K[:m, 0].max())[0]
                want, size = V[at].mean(0), np.abs(V[at]).mean(0)
                tol = size * (len(at) + 4) * 2.0 ** -24 + np.abs(want) * ps.U[np.dtype(dtype)] + ps.TINY[np.dtype(dtype)]
                for x in got[cu[b] + i, h * g:(h + 1) * g]:
                    ps.assert_within(x, want, tol)


FAR = [([1, 3], [0, 700]), ([6], [9000]), ([150], [0]), ([140, 2], [700, 3]), ([40], [9000])]


@pytest.mark.parametrize("down", [False, True])
@pytest.mark.parametrize("dtype,top", [(np.float16, 2048.0), (np.float16, 57344.0), (np.float32, 57344.0), (np.float32, 2.0 ** 40)])
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("batch", range(len(FAR)))
def test_scores_whose_multiples_of_the_scale_round_by_more_than_one(dtype, top, heads, down, batch):
    """up to 256 * 57344^2 / 16 = 5e10 in fp16: a step of fp32 is 4096 there"""
    largest_wins(*FAR[batch], *heads, dtype, top, down)


@pytest.mark.parametrize("top", [57344.0 * 2.0 ** 36, 57344.0 * 2.0 ** 41])
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("batch", range(len(FAR)))
def test_finite_scores_of_any_size_are_no_masked_ones(top, heads, batch):
    """fp32 scores of -1e32 and -1e35 and a sixteenth of them, nothing above"""
    largest_wins(*FAR[batch], *heads, np.float32, top, True)
