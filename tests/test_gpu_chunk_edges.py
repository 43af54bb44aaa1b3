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


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("batch", [([6], [1000]), ([6], [9000]), ([150], [700]), ([150, 3], [9000, 300]), ([300], [0]), ([1], [40])])
def test_infinities_reach_every_row_that_sees_them_whatever_they_weigh(dtype, heads, batch):
    """Values with infinities and NaN at keys of which half the rows hold the largest score so far and the others e^-300 of it, in
    places that all rows of a tile see and in places that some do not; early keys, whose weight is large until later ones come,
    among them.  A weight is never 0: the sum with such a value is what it is for any weight."""
    (n, start), (hq, hk, d) = batch, heads
    rng = np.random.default_rng(d)
    table, n_pages = ps.pages_for(n, start, rng)
    q = (0.5 * rng.standard_normal((sum(n), hq, d))).astype(dtype)
    q[..., 0] = 16 * (2 * rng.integers(0, 2, q.shape[:2]) - 1)     # the sign says which of the marked keys are far below
    k = rng.standard_normal((n_pages, hk, 128, d)).astype(dtype)
    k[..., 0] = 0
    v = rng.standard_normal(k.shape).astype(dtype)
    marked = {}                                                    # key: (dim, value)
    for b in range(len(n)):
        last = start[b] + n[b] - 1
        for i, key in enumerate(sorted({0, 3, 31, min(64, last), last // 3, last // 2, max(last - 70, 0), max(last - 2, 0), last})):
            if key > last:
                continue
            k[table[b, key // 128], :, key % 128, 0] = (1 if i % 2 else -1) * 300 / 16 * np.sqrt(d)
            v[table[b, key // 128], :, key % 128, 3 + i] = [np.inf, -np.inf, np.nan][i % 3]
            if i:
                v[table[b, key // 128], :, key % 128, 20] = np.inf if i != 4 else -np.inf
    k[..., 1] = q[..., 1] = 0
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, max(n), max(s + m for s, m in zip(start, n)))
    want, tol = ps.chunk_want(q, k, v, table, n, start, max(s + m for s, m in zip(start, n)))
    assert not np.isfinite(want).all() and np.isfinite(want).any()
    fine = np.isfinite(want)
    ps.assert_within(got, want, np.where(fine, tol, 0))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [6, 150])
def test_a_row_whose_scores_are_no_numbers_stays_one_without(dtype, n):
    """a NaN or an infinite score makes the whole row NaN, also where a value that it sees is infinite"""
    q, k, v, table = ps.picking([n], [900], 4, 2, 64, dtype)
    v[table[0, 0], :, 5, 7] = np.inf
    k[table[0, 0], :, 6, :] = np.nan
    assert np.isnan(ps.chunk(q, k, v, table, ps.cu_of([n]), [900], n, 900 + n)).all()
    k[table[0, 0], :, 6, :] = np.inf            # queries hold zeros, too: 0 * inf
    assert np.isnan(ps.chunk(q, k, v, table, ps.cu_of([n]), [900], n, 900 + n)).all()
    k[table[0, 0], :, 6, :] = 0
    q[...] = 1
    k[table[0, 0], 0, 6, 9] = np.inf            # a score of +inf in the first kv head
    got = ps.chunk(q, k, v, table, ps.cu_of([n]), [900], n, 900 + n)
    assert np.isnan(got[:, :2]).all() and np.all(got[:, 2:, 7] == np.inf) and np.isfinite(np.delete(got[:, 2:], 7, -1)).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n,start", [(6, 300), (150, 700), (6, 9000)])
def test_scores_of_minus_infinity(dtype, n, start):
    """such a key weighs nothing; a row that has no other comes out as zeros"""
    q, k, v, table = ps.picking([n], [start], 4, 2, 64, dtype)
    q[...] = 1
    k[...] = 0
    k[table[0], 0, :, 5] = -np.inf              # the first kv head: every key
    k[table[0, 1], 1, 3:90, 5] = -np.inf        # the second: some
    got = ps.chunk(q, k, v, table, ps.cu_of([n]), [start], n, start + n)
    assert np.all(got[:, :2] == 0)
    gone = np.arange(131, 218)
    sums, numbers = ps.picking_want(q[:, 2:], k[:, 1:], v[:, 1:], table, [n], [start], lambda b, m: np.setdiff1d(np.arange(m), gone))
    assert ps.picking_error(got[:, 2:], sums, numbers) <= 0.25


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("heads", [(9, 3, 64), (7, 1, 128), (2, 2, 256)])
def test_many_sequences_over_long_caches(dtype, heads):
    """more sequences than lanes whose tiles are cut: the search for a piece, and for the tile to merge, over several loads"""
    rng = np.random.default_rng(3)
    n, start = rng.integers(0, 4, 150), rng.integers(0, 3000, 150)
    n[77], n[140], start[3], start[149], n[149] = 90, 200, 15000, 9000, 2
    q, k, v, table = ps.picking(list(n), list(start), *heads, dtype)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 200, int((n + start).max()))
    assert ps.picking_error(got, *ps.picking_want(q, k, v, table, n, start)) <= 0.25


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("max_len", [4097, 4224, 5000])
def test_max_len_of_a_cut_tile(dtype, max_len):
    """tokens behind max_len see the keys before it"""
    n, start = [300, 2], [4000, 8000]
    q, k, v, table = ps.picking(n, start, 4, 2, 128, dtype)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 300, max_len)
    sums, numbers = ps.picking_want(q, k, v, table, n, start, lambda b, m: np.arange(min(m, max_len)))
    assert ps.picking_error(got, sums, numbers) <= 0.25


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_captured_calls_follow_what_is_cut(dtype):
    """one graph, replayed over lengths whose tiles are cut and over others whose are not, of few rows and of many"""
    from axono_amd import HIPGraph, Tensor, libaxono as L

    def hip(a):
        return Tensor.from_numpy_ref(np.ascontiguousarray(a)).to("hip:0")

    T, B, hq, hk, d, longest = 120, 3, 4, 2, 64, 9200
    lots = [([1, 1, 1], [9000, 20, 300]), ([110, 4, 1], [0, 9100, 64]), ([0, 120, 0], [5, 0, 7]), ([2, 90, 3], [700, 9000, 0]), ([1, 0, 1], [0, 0, 127])]
    at = [hip(np.zeros(s, t)) for s, t in (((T, hq, d), dtype), ((230, hk, 128, d), dtype), ((230, hk, 128, d), dtype), ((B, 73), np.int32),
                                           ((B + 1,), np.int32), ((B,), np.int32))]
    g, out = HIPGraph(), []
    g.capture(lambda: out.append(L.chunk_attention_paged(*at, T, longest)))
    for seed in (0, 1):
        for n, start in lots:
            q, k, v, table = ps.picking(n, start, hq, hk, d, dtype, seed)
            wide = np.full((B, 73), -1, np.int32)
            wide[:, :table.shape[1]] = table
            pool = np.full((2, 230, hk, 128, d), np.nan, dtype)     # (NaN where no sequence has a page)
            pool[0, :len(k)], pool[1, :len(v)] = k, v
            rows = np.zeros((T, hq, d), dtype)
            rows[:len(q)] = q
            for a, x in zip(at, (rows, pool[0], pool[1], wide, ps.cu_of(n), np.array(start, np.int32))):
                a.copy_from_numpy(x)
            g.replay()
            got = out[-1].numpy()[:len(q)]
            assert ps.picking_error(got, *ps.picking_want(q, k, v, table, n, start)) <= 0.25, (n, start)
            eager = L.chunk_attention_paged(*at, T, longest)
            np.testing.assert_array_equal(eager.numpy()[:len(q)].view(np.uint8), got.view(np.uint8))


@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("batch", [([1], [41]), ([6], [300]), ([150], [100]), ([3], [9000])])
def test_finite_values_near_the_end_of_fp32(heads, batch):
    """a row's weighted mean of values up to 3e35 .. 1e37 is finite wherever the sum of weights of at most 1 times them is: 3.4e38 over
    the number of keys.  Scores rise by 5 on the way, so that what is summed first was the largest then."""
    (n, start), (hq, hk, d) = batch, heads
    rng = np.random.default_rng(1)
    table, n_pages = ps.pages_for(n, start, rng)
    keys = start[0] + n[0]
    q, k = np.zeros((n[0], hq, d), np.float32), np.zeros((n_pages, hk, 128, d), np.float32)
    q[..., 0] = 8
    for key in range(keys):                     # in steps of a fifth of what the first token sees
        k[table[0, key // 128], :, key % 128, 0] = np.sqrt(d) / 8 * min(5 * key // (start[0] + 1), 5)
    v = (rng.uniform(0.5, 1, k.shape) * 3.4e38 / keys * 0.9).astype(np.float32)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, n[0], keys)
    want, tol = ps.chunk_want(q, k, v, table, n, start, keys)
    assert np.isfinite(want).all()
    ps.assert_within(got, want, tol)


@pytest.mark.parametrize("batch", [([1], [41]), ([150], [100]), ([3], [9000])])
def test_finite_values_near_nothing(batch):
    """values of 1e-37: a weight of 2^-8 makes a product denormal, off by 2^-150, the mean by 2^-142 (and its own rounding)"""
    n, start = batch
    rng = np.random.default_rng(2)
    table, n_pages = ps.pages_for(n, start, rng)
    q, k = np.zeros((n[0], 4, 64), np.float32), np.zeros((n_pages, 2, 128, 64), np.float32)
    v = rng.uniform(0.5e-37, 1e-37, k.shape).astype(np.float32)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, n[0], start[0] + n[0])
    want, tol = ps.chunk_want(q, k, v, table, n, start, start[0] + n[0])
    ps.assert_within(got, want, tol + 2.0 ** -141)
