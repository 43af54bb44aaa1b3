"""Penalties, biases and masks on logits, against 64 bits."""
import numpy as np
import pytest

import paged_step_util as ps

pytestmark = pytest.mark.gpu


def make(B, V, H, bias, mask, dtype, ids, seed=0):
    rng = np.random.default_rng(seed)
    x = (4 * rng.standard_normal((B, V))).astype(dtype)
    hist = rng.integers(-2, max(V // 3, 2), (B, H)).astype(ids) if H else None
    if H:
        hist[:, H // 2] = V + 5                     # an id outside the vocabulary
        hist[:, 0] = V - 1
    n = rng.integers(0, H + 1, B) if H else None
    prompt = n // 2 if H else None
    rep, pres, freq = (rng.uniform(a, b, B).astype(np.float32) for a, b in ((0.8, 1.5), (-1, 1), (-0.2, 0.5)))
    bi = rng.integers(-1, V + 1, (B, bias)).astype(np.int32) if bias else None
    bv = rng.uniform(-5, 5, (B, bias)).astype(np.float32) if bias else None
    if bias > 2:
        bi[:, 2] = bi[:, 0]                         # the same id twice
    al = rng.integers(0, 1 << 32, (B, (V + 31) // 32), np.uint64).astype(np.uint32) if mask else None
    return x, hist, n, prompt, rep, pres, freq, bi, bv, al


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B,V,H,bias,mask,ids,by_step", [
    (1, 1, 1, 0, False, np.int32, False), (1, 1, 0, 1, True, np.int32, False), (3, 1000, 50, 7, True, np.int64, True),
    (2, 2047, 300, 0, False, np.int32, False), (5, 2049, 64, 300, True, np.int32, True), (1, 151936, 700, 8, True, np.int32, False),
    (4, 40000, 5000, 65, True, np.int64, False), (70, 4096, 129, 3, True, np.int64, True), (2, 5000, 20000, 4, True, np.int32, False),
    (2, 70001, 16384, 0, True, np.int64, True)])
def test_logits(dtype, B, V, H, bias, mask, ids, by_step):
    args = make(B, V, H, bias, mask, dtype, ids)
    want, tol = ps.logits_want(*args)
    ps.assert_within(ps.logits(*args, by_step=by_step), want, tol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("stride", [4096, 4099, 5000])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_in_place(dtype, stride, in_place):
    args = make(6, 4096, 90, 5, True, dtype, np.int32)
    want, tol = ps.logits_want(*args)
    ps.assert_within(ps.logits(*args, stride=stride, in_place=in_place), want, tol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_untouched_logits_keep_their_bits(dtype):
    x, hist, n, prompt, rep, pres, freq, bi, bv, al = make(3, 9001, 40, 6, True, dtype, np.int32)
    none = (None,) * 9
    np.testing.assert_array_equal(ps.logits(x, *none), x)
    got = ps.logits(x, hist, n, prompt, rep, pres, freq, bi, bv, None)
    free = np.ones(x.shape, bool)
    for b in range(3):
        free[b, hist[b, :n[b]][(hist[b, :n[b]] >= 0) & (hist[b, :n[b]] < 9001)]] = False
        free[b, bi[b][(bi[b] >= 0) & (bi[b] < 9001)]] = False
    np.testing.assert_array_equal(got[free], x[free])


def test_each_part_alone_and_missing_lengths():
    x, hist, n, prompt, rep, pres, freq, bi, bv, al = make(4, 3001, 80, 9, True, np.float32, np.int64)
    full, zero = np.full(4, 80), np.zeros(4, int)
    for a in ((rep, None, None), (None, pres, None), (None, None, freq)):
        want, tol = ps.logits_want(x, hist, full, zero, *a, None, None, None)
        ps.assert_within(ps.logits(x, hist, None, None, *a, None, None, None), want, tol)
    want, tol = ps.logits_want(x, None, None, None, None, None, None, bi, bv, None)
    ps.assert_within(ps.logits(x, None, None, None, None, None, None, bi, bv, None), want, tol)


def test_lengths_outside_the_history_are_clamped():
    x, hist, _, _, rep, pres, freq, _, _, _ = make(3, 500, 30, 0, False, np.float32, np.int32)
    want, tol = ps.logits_want(x, hist, [0, 30, 30], [0, 30, 0], rep, pres, freq, None, None, None)
    ps.assert_within(ps.logits(x, hist, [-4, 99, 30], [5, 200, -3], rep, pres, freq, None, None, None), want, tol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_special_values_and_empty_masks(dtype):
    x = np.zeros((2, 64), dtype)
    x[0, :5] = [np.inf, -np.inf, np.nan, 0.0, -0.0]
    hist = np.array([[0, 1, 2, 3, 4, 4], [1, 1, 1, 1, 1, 1]], np.int32)
    rep, pres, freq = np.array([2, 2], np.float32), np.array([.5, .5], np.float32), np.array([.25, .25], np.float32)
    allowed = np.array([[0xffffffff] * 2, [0, 0]], np.uint32)
    got = ps.logits(x, hist, [6, 6], [0, 3], rep, pres, freq, None, None, allowed).astype(np.float64)
    np.testing.assert_array_equal(got[0, :6], [np.inf, -np.inf, np.nan, -0.75, -1.0, 0.0])
    assert np.all(got[1] == -np.inf)                # a row whose mask allows nothing


def test_a_count_beyond_sixteen_bits():
    hist = np.zeros((1, 70000), np.int32)
    x = np.zeros((1, 300), np.float32)
    got = ps.logits(x, hist, [70000], [0], None, None, np.array([1.0], np.float32), None, None, None)
    assert got[0, 0] == -70000.0 and np.all(got[0, 1:] == 0)


def test_then_argmax_picks_among_the_allowed():
    rng = np.random.default_rng(8)
    B, V = 16, 151936
    x = rng.standard_normal((B, V)).astype(np.float32)
    allowed = np.zeros((B, V // 32), np.uint32)
    only = rng.integers(0, V, (B, 3))
    for b in range(B):
        for t in only[b]:
            allowed[b, t // 32] |= np.uint32(1 << (t % 32))
    y = ps.logits(x, None, None, None, None, None, None, None, None, allowed)
    dy, ids = ps.dev(y), ps.DeviceBuffer(B * 8)
    ps.check(ps.lib().axhip_argmax(dy.ptr, ids.ptr, ps.F32, B, V, None), "argmax")
    got = ids.download(np.int64, (B,))
    assert [int(g) for g in got] == [int(max(sorted(only[b]), key=lambda t: x[b, t])) for b in range(B)]
