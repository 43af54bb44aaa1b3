"""Attention of a ragged batch of new tokens over a paged cache, against 64 bits."""
import numpy as np
import pytest

import paged_step_util as ps

pytestmark = pytest.mark.gpu


def make(n, start, hq, hk, d, dtype, seed=0, rows_behind=0, scale=1.0):
    rng = np.random.default_rng(seed)
    table, n_pages = ps.pages_for(n, start, rng)
    T = sum(n) + rows_behind
    q = (scale * rng.standard_normal((T, hq, d))).astype(dtype)
    pools = [rng.standard_normal((n_pages, hk, 128, d)).astype(dtype) for _ in range(2)]
    return q, pools[0], pools[1], table


def run(n, start, hq, hk, d, dtype, seed=0, max_len=None, scale=1.0, max_q=None):
    q, k, v, table = make(n, start, hq, hk, d, dtype, seed, scale=scale)
    max_len = max(max(s + m for s, m in zip(start, n)), 0) if max_len is None else max_len
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, max(n) if max_q is None else max_q, max_len)
    want, tol = ps.chunk_want(q, k, v, table, n, start, max_len)
    ps.assert_within(got, want, tol)


SHAPES = [(16, 8, 128), (32, 8, 128), (4, 4, 64), (8, 1, 64), (2, 1, 256), (3, 1, 128), (20, 2, 64), (64, 1, 128)]
BATCHES = [
    ([1], [0]),                                     # one token, one key
    ([1], [127]), ([1], [128]),                     # a page's last and first row
    ([2, 1, 3], [0, 1000, 254]),
    ([1] * 5, [0, 1, 31, 32, 700]),                 # decode
    ([4] * 4, [2047, 60, 0, 900]),                  # drafts
    ([33, 0, 1, 17], [5, 9, 2000, 111]),            # mixed, one without tokens
    ([129, 64], [0, 65]),
    ([300], [77]),
]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("batch", range(len(BATCHES)))
def test_chunk_attention(dtype, shape, batch):
    n, start = BATCHES[batch]
    run(n, start, *shape, dtype, seed=batch)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_many_sequences(dtype):
    """more sequences than lanes, some without tokens: the search for a workgroup's tile runs over several loads"""
    rng = np.random.default_rng(9)
    n = rng.integers(0, 4, 150)
    start = rng.integers(0, 400, 150)
    run(list(n), list(start), 4, 2, 64, dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [1, 16, 40, 70])
def test_long_cache_is_cut_into_pieces(dtype, n):
    run([n, 1], [9000, 3], 4, 2, 128, dtype, seed=n)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_large_scores(dtype):
    """scores far apart: the running maximum moves late and often"""
    run([70, 3], [200, 500], 4, 2, 64, dtype, scale=12.0)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rows_without_keys_are_zeros(dtype):
    n, start = [5, 40, 3], [-3, -40, 0]
    q, k, v, table = make(n, [0, 0, 0], 4, 2, 64, dtype)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 40, 100)
    want, tol = ps.chunk_want(q, k, v, table, n, start, 100)
    assert np.all(got[:3] == 0) and np.all(got[5:45] == 0) and np.all(got[3:5] != 0)
    ps.assert_within(got, want, tol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_max_len_and_max_q_bound_what_is_done(dtype):
    run([200, 4], [100, 290], 4, 2, 64, dtype, max_len=256)
    n, start = [50, 3], [10, 700]
    q, k, v, table = make(n, start, 4, 2, 64, dtype)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 20, 703)
    want, tol = ps.chunk_want(q, k, v, table, n, start, 703)
    ps.assert_within(got[:20], want[:20], tol[:20])
    ps.assert_within(got[50:], want[50:], tol[50:])
    assert np.all(got[20:50] == 9.0)                # more tokens than max_q: left as they were


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rows_behind_the_last_sequence_stay(dtype):
    n, start = [3, 70], [128, 0]
    q, k, v, table = make(n, start, 4, 2, 128, dtype, rows_behind=5)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 70, 131)
    want, tol = ps.chunk_want(q[:73], k, v, table, n, start, 131)
    ps.assert_within(got[:73], want, tol)
    assert np.all(got[73:] == 9.0)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [6, 150])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, d, n):
    """NaN behind the last key, infinities and NaN in keys and values of later tokens"""
    start = 130
    q, k, v, table = make([n], [start], 4, 2, d, dtype)
    end = start + n
    for pool in (k, v):
        pool[table[0, (end - 1) // 128], :, end % 128 if end % 128 else 128:] = np.nan
    free = [p for p in range(k.shape[0]) if p not in table[0]]
    k[free], v[free] = np.nan, np.inf
    row = lambda pool, key: pool[table[0, key // 128], :, key % 128]  # noqa: E731
    row(v, end - 1)[:, 5] = np.nan
    row(v, end - 2)[:, 9] = np.inf
    row(v, end - 3)[:, 11] = -np.inf
    row(k, end - 1)[1, 3] = np.nan                  # only the last token sees this key
    got = ps.chunk(q, k, v, table, ps.cu_of([n]), [start], n, end)
    want, tol = ps.chunk_want(q, k, v, table, [n], [start], end)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)) and fine[:-3].all() and not fine[-1, 2:].any()
    ps.assert_within(np.where(fine, got, 0), np.where(fine, want, 0), np.where(fine, tol, 0))
    assert np.all(got[-2:, :2, 9] == np.inf) and np.all(got[-3:-1, :, 11] == -np.inf)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_infinity_among_the_keys_that_all_see_of_a_cut_tile(dtype):
    n, start = [20], [6000]
    q, k, v, table = make(n, start, 4, 2, 64, dtype)
    v[table[0, 10], 0, 3, 7] = np.inf
    v[table[0, 46], 1, 6018 % 128, 2] = -np.inf     # key 6018: seen by the last two tokens
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 20, 6020)
    want, tol = ps.chunk_want(q, k, v, table, n, start, 6020)
    ps.assert_within(got, want, tol)


def test_bad_pages_stay_inside_the_pool():
    """page numbers outside the pool are clamped: wrong values, no access outside; sequences with good pages are right"""
    n, start = [4, 4], [300, 300]
    q, k, v, table = make(n, start, 4, 2, 64, np.float16)
    table[0] = [-7, 1 << 30, k.shape[0]]
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 4, 304)
    want, tol = ps.chunk_want(q, k, v, table, n, start, 304)    # (the same clamp)
    ps.assert_within(got, want, tol)


def test_same_bits_again_and_with_another_workspace():
    n, start = [60, 1, 7], [3000, 5000, 0]
    q, k, v, table = make(n, start, 8, 2, 128, np.float16)
    a = ps.chunk(q, k, v, table, ps.cu_of(n), start, 60, 5001)
    for dirty in (True, False):
        np.testing.assert_array_equal(a, ps.chunk(q, k, v, table, ps.cu_of(n), start, 60, 5001, dirty=dirty))


def test_agrees_with_decode_attention_over_the_same_pages():
    n, start = [1] * 6, [0, 5, 127, 128, 1000, 2500]
    q, k, v, table = make(n, start, 16, 8, 128, np.float16)
    got = ps.chunk(q, k, v, table, ps.cu_of(n), start, 1, 2501)
    bufs = [ps.dev(a) for a in (q, k, v, table, np.array(start, np.int32) + 1)]
    out = ps.DeviceBuffer(q.nbytes)
    size = ps.lib().axhip_gqa_decode_workspace_bytes(6, 16, 8, 128, 2501)
    ws = ps.DeviceBuffer(max(size, 256))
    ps.check(ps.lib().axhip_gqa_decode_paged(*[b.ptr for b in bufs], out.ptr, ws.ptr, ws.nbytes, ps.F16, 6, 16, 8, 128, 2501,
                                             table.shape[1], k.shape[0], None), "gqa_decode_paged")
    want, tol = ps.chunk_want(q, k, v, table, n, start, 2501)
    ps.assert_within(got, want, tol)
    assert np.all(np.abs(got.astype(float) - out.download(np.float16, q.shape).astype(float)) <= 2 * tol)


def test_agrees_with_prefill_attention_of_the_dense_cache():
    S, hq, hk, d = 200, 4, 2, 64
    q, k, v, table = make([S], [0], hq, hk, d, np.float16)
    got = ps.chunk(q, k, v, table, ps.cu_of([S]), [0], S, S)
    dense = [p[table[0]].transpose(1, 0, 2, 3).reshape(1, hk, -1, d) for p in (k, v)]
    dq, dk, dv, out = ps.dev(q), ps.dev(dense[0]), ps.dev(dense[1]), ps.DeviceBuffer(q.nbytes)
    ps.check(ps.lib().axhip_prefill_attention(dq.ptr, dk.ptr, dv.ptr, None, out.ptr, ps.F16, 1, S, hq, hk, d, dense[0].shape[2], None),
             "prefill_attention")
    _, tol = ps.chunk_want(q, k, v, table, [S], [0], S)
    assert np.all(np.abs(got.astype(float) - out.download(np.float16, q.shape).astype(float)) <= 2 * tol)


def test_many_small_weights_add_up():
    """A row whose first key has score 17.5 and its 65535 others 0: each of these weighs e^-17.5 = 2^-25.2, together 2^-9.2.  256 x 2
    tiles over the same pages fill the device, so that most of a row's keys are taken in one piece.  The result is
    N e^-17.5 / (1 + N e^-17.5) to the rounding of such a weight, 2^-25 / 2^-15.3 at 2^10 for the largest, and of the result."""
    B, hk, keys = 256, 2, 65536
    k, v = (np.zeros((keys // 128, hk, 128, 64), np.float16) for _ in range(2))
    v[...] = 1
    k[0, :, 0, 0], v[0, :, 0] = 17.5, 0
    q = np.zeros((B, hk, 64), np.float16)
    q[..., 0] = 8
    table = np.tile(np.arange(keys // 128, dtype=np.int32), (B, 1))
    got = ps.chunk(q, k, v, table, ps.cu_of([1] * B), [keys - 1] * B, 1, keys).astype(np.float64)
    rest = (keys - 1) * np.exp(-17.5)
    want = rest / (1 + rest)
    assert np.abs(got / want - 1).max() <= 2.0 ** -9.7 + 2.0 ** -11 + 2.0 ** -17
