"""The check of chunk attention by whole numbers sees a single wrong key: mistakes planted in the oracle, on the CPU."""
import numpy as np
import pytest

import paged_step_util as ps


def off(dtype, n, start, keys_of, d=64, hk=2):
    q, k, v, table = ps.picking(n, start, 4, hk, d, dtype, seed=3)
    sums, numbers = ps.picking_want(q, k, v, table, n, start)
    bad_sums, bad_numbers = ps.picking_want(q, k, v, table, n, start, keys_of)
    got = (bad_sums / bad_numbers[..., None]).astype(dtype)
    return ps.picking_error(got, sums, numbers)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_right_results_pass(dtype):
    assert off(dtype, [5, 1], [9000, 77], None) <= 0.25
    assert off(dtype, [1], [0], None) <= 0.25


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("key", [0, 31, 32, 63, 64, 127, 128, 4095, 4608, 8959, 9000, 9001])
def test_one_key_left_out_or_taken_twice(dtype, key):
    """(some head of the last row picks the key)"""
    n, start = [2], [9000]
    assert off(dtype, n, start, lambda b, m: np.delete(np.arange(m), min(key, m - 1))) > 0.5
    assert off(dtype, n, start, lambda b, m: np.append(np.arange(m), min(key, m - 1))) > 0.5


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_blocks_and_borders(dtype):
    n, start = [2], [9000]
    mistakes = [lambda m: np.r_[0:4608, 4640:m],        # a block of 32 keys
                lambda m: np.r_[0:4608, 4672:m],        # a stage of 64
                lambda m: np.r_[0:4608, 4736:m],        # a page
                lambda m: np.arange(m + 1),             # the next token's key
                lambda m: np.arange(m - 1),             # not its own
                lambda m: np.r_[0:4640, 4608:4640, 4640:m],
                lambda m: np.r_[0:4608, 4096:4128, 4640:m]]  # another block's keys
    for keys in mistakes:
        assert off(dtype, n, start, lambda b, m: keys(m)) > 0.5
