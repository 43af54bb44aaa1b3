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
