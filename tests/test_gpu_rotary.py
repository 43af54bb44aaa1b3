"""Rotation by a frequency table, alone and on the way into a paged cache, against 64 bits."""
import numpy as np
import pytest

import paged_step_util as ps

pytestmark = pytest.mark.gpu


def table(rd, theta=1e6):
    return (theta ** (-np.arange(0, rd, 2) / rd)).astype(np.float32)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,hq,hk,d,rd", [
    (1, 1, 1, 8, 2), (1, 16, 8, 128, 128), (3, 5, 1, 64, 32), (7, 4, 2, 80, 20), (5, 3, 3, 80, 40), (33, 16, 8, 128, 64),
    (2, 2, 2, 96, 24), (9, 7, 1, 256, 256), (4, 2, 1, 512, 512), (4, 2, 1, 512, 6), (300, 8, 4, 128, 32), (17, 1, 0, 64, 62)])
def test_rotary(dtype, interleaved, rows, hq, hk, d, rd):
    rng = np.random.default_rng(rows * d + rd)
    q = rng.standard_normal((rows, hq, d)).astype(dtype)
    k = rng.standard_normal((rows, hk, d)).astype(dtype) if hk else None
    pos = rng.integers(-5, 1 << 20, rows)
    f = table(rd)
    got = ps.rotary_qk(q, k, pos, f, 1.25, interleaved, rd)
    for x, y in zip((q, k), got):
        if x is None:
            continue
        want, size = ps.turned(x, pos, f, rd, interleaved, 1.25)
        ps.assert_within(y, want, size * ps.ROTATION + np.abs(want) * ps.U[x.dtype] + ps.TINY[x.dtype])
        np.testing.assert_array_equal(y[..., rd:], x[..., rd:])   # the rest of the head is copied


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved,qs,ks", [(False, 3 * 64 + 1, 64 + 3), (False, 3 * 64 + 2, 64 + 4), (True, 3 * 64 + 2, 64 + 6), (True, 256, 128)])
def test_rotary_row_strides(dtype, interleaved, qs, ks):
    rng = np.random.default_rng(qs)
    q, k = rng.standard_normal((6, 3, 64)).astype(dtype), rng.standard_normal((6, 1, 64)).astype(dtype)
    pos, f = rng.integers(0, 5000, 6), table(48)
    for x, y in zip((q, k), ps.rotary_qk(q, k, pos, f, 1.0, interleaved, 48, qs, ks)):
        want, size = ps.turned(x, pos, f, 48, interleaved, 1.0)
        ps.assert_within(y, want, size * ps.ROTATION + np.abs(want) * ps.U[x.dtype] + ps.TINY[x.dtype])


def test_rotary_far_positions_keep_their_angle():
    """fp32 angles are off by pos 2^-24 radians; here the angle stays exact at any position"""
    rng = np.random.default_rng(0)
    q = rng.standard_normal((4, 2, 128)).astype(np.float32)
    pos, f = np.array([(1 << 31) + 12345, 1 << 40, -(1 << 33), 0]), table(128)
    want, size = ps.turned(q, pos, f, 128, False, 1.0)
    got, _ = ps.rotary_qk(q, None, pos, f, 1.0, False, 128)
    ps.assert_within(got, want, size * (ps.ROTATION + 2.0 ** 40 * 2.0 ** -52))   # (the product itself is in 64 bits)
    np.testing.assert_array_equal(got[3], q[3])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_negated_positions_are_the_gradient(interleaved):
    """d(sum w y)/dx is the rotation of w at negated positions: against differences of the formula in 64 bits"""
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((2, 1, 16)).astype(np.float32), rng.standard_normal((2, 1, 16)).astype(np.float32)
    pos, f = np.array([5, 1000]), table(12)
    got, _ = ps.rotary_qk(w, None, -pos, f, 1.5, interleaved, 12)
    grad = np.zeros(x.shape)
    for at in np.ndindex(*x.shape):
        e = np.zeros(x.shape)
        e[at] = 1e-3
        up, _ = ps.turned(x + e, pos, f, 12, interleaved, 1.5)
        down, _ = ps.turned(x - e, pos, f, 12, interleaved, 1.5)
        grad[at] = ((up - down) / 2e-3 * w).sum()
    _, size = ps.turned(w, -pos, f, 12, interleaved, 1.5)
    ps.assert_within(got, grad, size * ps.ROTATION + np.abs(grad) * 2.0 ** -24 + 1e-9)


def test_rotary_in_place_and_special_values():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((40, 6, 128)).astype(np.float32)
    x[3, 2, 100] = np.inf      # behind the rotated part
    x[4, 1, 127] = np.nan
    x[5, 0, 3] = np.inf        # inside: its pair turns into what IEEE makes of it, nothing else
    pos, f = rng.integers(0, 4096, 40), table(64)
    dx, dp, df = ps.dev(x), ps.dev(pos), ps.dev(f)
    ps.check(ps.lib().axhip_rotary_qk(dx.ptr, 6 * 128, None, 0, dp.ptr, df.ptr, 1.0, 0, 64, dx.ptr, None, ps.F32, 40, 6, 0, 128, None),
             "rotary_qk")
    got = dx.download(np.float32, x.shape)
    want, size = ps.turned(x, pos, f, 64, False, 1.0)
    touched = np.zeros(x.shape, bool)
    touched[5, 0, [3, 35]] = True
    assert not np.isfinite(got[touched]).any()
    np.testing.assert_array_equal(got[..., 64:], x[..., 64:])
    ps.assert_within(np.where(touched, 0, got), np.where(touched, 0, want),
                     np.where(np.isfinite(size), size, 0) * ps.ROTATION + np.where(np.isfinite(want), np.abs(want), 0) * 2.0 ** -24)


def test_more_rows_than_one_launch_takes():
    rows = (1 << 25) + 70
    x = np.tile(np.arange(1, 57, dtype=np.float16).reshape(7, 1, 8) / 8, (rows // 7 + 1, 1, 1))[:rows]
    pos, f = np.arange(rows, dtype=np.int64) % 1000, table(8)
    dx, dp, df = ps.dev(x), ps.dev(pos), ps.dev(f)
    ps.check(ps.lib().axhip_rotary_qk(dx.ptr, 8, None, 0, dp.ptr, df.ptr, 1.0, 0, 8, dx.ptr, None, ps.F16, rows, 1, 0, 8, None), "rotary_qk")
    got = dx.download(np.float16, x.shape)
    for at in (slice(0, 200), slice((1 << 25) - 100, rows)):
        want, size = ps.turned(x[at], pos[at], f, 8, False, 1.0)
        ps.assert_within(got[at], want, size * ps.ROTATION + np.abs(want) * 2.0 ** -11 + 2.0 ** -25)


# ---- append ------------------------------------------------------------------------------------------------------------
CASES = [
    # n, start, hq, hk, d, rd, interleaved, norm, axes
    ([1], [0], 2, 1, 64, 64, False, True, 1),
    ([1, 1, 1], [127, 128, 5000], 16, 8, 128, 128, False, True, 3),
    ([5, 0, 1, 130], [125, 7, 300, 0], 4, 2, 128, 64, True, False, 1),
    ([3, 2], [-2, 250], 3, 3, 256, 64, False, True, 1),       # a negative start: those rows go nowhere
    ([70] + [1] * 70 + [0] * 3, [0] + list(range(70)) + [9, 9, 9], 2, 2, 64, 16, True, True, 3),
    ([2, 3], [0, 126], 1, 1, 80, 20, False, True, 1),
    ([4], [100], 7, 1, 96, 2, True, False, 3),
]


@pytest.mark.parametrize("types", [(np.float32, np.float16), (np.float16, np.float16), (np.float32, np.float32), (np.float16, np.float32)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append(case, types):
    n, start, hq, hk, d, rd, interleaved, norm, axes = CASES[case]
    rng = np.random.default_rng(case)
    T = sum(n)
    table_, n_pages = ps.pages_for(n, start, rng)
    qkv = rng.standard_normal((T, hq + 2 * hk, d)).astype(types[0])
    wt = np.float16 if case % 2 else np.float32
    w = [(1 + 0.1 * rng.standard_normal(d)).astype(wt) for _ in range(2)] if norm else [None, None]
    pools = [rng.standard_normal((n_pages, hk, 128, d)).astype(types[1]) for _ in range(2)]
    pos = rng.integers(0, 9000, (axes, T))
    sec = (rd // 6, rd // 8)
    f = table(rd)
    args = (hq, hk, w, 1e-6, norm)
    got = ps.append(qkv, *args, pos, axes, f, 1.1, interleaved, rd, sec, ps.cu_of(n), start, table_, *pools)
    want, tol = ps.append_want(qkv, *args, pos, f, 1.1, interleaved, rd, ps.mrope_axis(rd, *sec) if axes == 3 else None, n, start,
                               table_, *pools)
    for g, x, e in zip(got, want, tol):
        ps.assert_within(g, x, e)


def test_append_takes_the_key_position_without_positions():
    rng = np.random.default_rng(1)
    n, start = [3, 1], [126, 40]
    table_, n_pages = ps.pages_for(n, start, rng)
    qkv = rng.standard_normal((4, 4, 64)).astype(np.float32)
    pools = [np.zeros((n_pages, 1, 128, 64), np.float16) for _ in range(2)]
    f = table(64)
    args = (2, 1, [None, None], 1e-6, True)
    got = ps.append(qkv, *args, None, 1, f, 1.0, False, 64, (0, 0), ps.cu_of(n), start, table_, *pools)
    want, tol = ps.append_want(qkv, *args, np.array([126, 127, 128, 40]), f, 1.0, False, 64, None, n, start, table_, *pools)
    for g, x, e in zip(got, want, tol):
        ps.assert_within(g, x, e)


def test_append_leaves_alone_what_is_not_a_sequences():
    """rows behind the last sequence, pages outside the pool, positions behind the table: nothing is read or written there"""
    rng = np.random.default_rng(2)
    n, start = [2, 2, 1], [127, 500, 3]                     # the second sequence runs behind its table
    table_ = np.array([[4, -1], [2, 1], [1 << 30, 0]], np.int32)
    qkv = rng.standard_normal((9, 6, 64)).astype(np.float32)  # 4 rows belong to nobody
    pools = [rng.standard_normal((5, 2, 128, 64)).astype(np.float16) for _ in range(2)]
    f, pos = table(64), rng.integers(0, 100, (1, 9))
    args = (2, 2, [None, None], 1e-6, False)
    got = ps.append(qkv, *args, pos, 1, f, 1.0, False, 64, (0, 0), ps.cu_of(n), start, table_, *pools)
    want, tol = ps.append_want(qkv[:5], *args, pos[:, :5], f, 1.0, False, 64, None, n, start, table_, *pools)
    ps.assert_within(got[0][:5], want[0], tol[0])
    assert np.all(got[0][5:] == 9.0)
    for g, x, e in zip(got[1:], want[1:], tol[1:]):
        ps.assert_within(g, x, e)
    assert np.count_nonzero(got[1] != pools[0]) <= 2 * 64   # one row of one page


def test_append_same_bits_as_rotary_and_copy():
    """append without norm = axhip_rotary_qk and a byte copy of v"""
    rng = np.random.default_rng(4)
    n, start = [140], [60]
    table_, n_pages = ps.pages_for(n, start, rng)
    qkv = rng.standard_normal((140, 12, 128)).astype(np.float16)
    pools = [np.zeros((n_pages, 4, 128, 128), np.float16) for _ in range(2)]
    pos, f = rng.integers(0, 30000, (1, 140)), table(128)
    q, kp, vp = ps.append(qkv, 4, 4, [None, None], 1e-6, False, pos, 1, f, 1.0, True, 128, (0, 0), ps.cu_of(n), start, table_, *pools)
    wq, wk = ps.rotary_qk(qkv[:, :4], qkv[:, 4:8], pos[0], f, 1.0, True, 128)
    at = 60 + np.arange(140)
    np.testing.assert_array_equal(q, wq)
    np.testing.assert_array_equal(kp[table_[0, at // 128], :, at % 128], wk)
    np.testing.assert_array_equal(vp[table_[0, at // 128], :, at % 128], qkv[:, 8:])


@pytest.mark.parametrize("append", [False, True])
def test_cosine_and_sine_are_those_of_the_angle_in_64_bits(append):
    """(1, 0) turns into cosine and sine: half a step of the value from each of two roundings, a step of sincosf; below 1 a step is
    2^-24 at most.  An angle near pi cut to 32 bits is off by 2^-23 alone."""
    rng = np.random.default_rng(12)
    d, T = 128, 2000
    pos, f = rng.integers(0, 1 << 20, T), table(d, 1e4)
    x = np.zeros((T, 2, d), np.float32)
    x[..., :d // 2] = 1
    if append:
        qkv = np.concatenate([x, x[:, :2]], axis=1)
        table_, n_pages = ps.pages_for([T], [0], rng)
        pools = [np.zeros((n_pages, 1, 128, d), np.float32) for _ in range(2)]
        got, _, _ = ps.append(qkv, 2, 1, [None, None], 1e-6, False, pos[None], 1, f, 1.0, False, d, (0, 0), ps.cu_of([T]), [0], table_, *pools)
    else:
        got, _ = ps.rotary_qk(x, None, pos, f, 1.0, False, d)
    want, _ = ps.turned(x, pos, f, d, False, 1.0)
    assert np.abs(got.astype(np.float64) - want).max() <= 2 * 2.0 ** -24
