"""Host page tables and lengths of narrow integer types are checked as the numbers they hold."""

from __future__ import annotations

import numpy as np
import pytest
from tests.test_cpu_serving_ops import _pool, _t


@pytest.mark.parametrize("dtype", [np.uint8, np.int8, np.int16, np.uint32, np.uint64])
def test_lengths_near_the_types_limit_do_not_wrap(dtype):
    from tensorgrad_b200.ops import append_pages

    top = min(int(np.iinfo(dtype).max), 1 << 20)
    pool = _pool(shape=(2, 1, 4, 8))
    pages = -(-top // 4)  # room for `top` positions, not for ten more
    table = np.zeros((1, pages), np.int64)
    k = _t((1, 1, 10, 8))
    with pytest.raises(IndexError, match="lengths must be in"):
        append_pages(k, k, pool, pool, table, np.array([top], dtype))


def test_pages_about_to_be_written_are_checked_behind_narrow_lengths():
    from tensorgrad_b200.ops import append_pages

    pool = _pool(shape=(2, 1, 4, 8))
    table = np.zeros((1, 80), np.int64)
    table[0, 64] = 2  # the page of positions 256 to 259, which is not in the pool
    k = _t((1, 1, 10, 8))
    with pytest.raises(IndexError, match="page ids"):
        append_pages(k, k, pool, pool, table, np.array([250], np.uint8))


def test_more_new_tokens_than_the_lengths_type_holds():
    from tensorgrad_b200.ops import append_pages

    pool = _pool(shape=(2, 1, 4, 8))
    k = _t((1, 1, 300, 8))
    with pytest.raises(IndexError, match="lengths must be in"):
        append_pages(k, k, pool, pool, np.zeros((1, 80), np.uint8), np.array([100], np.uint8))


def test_ids_beyond_64_bits_of_sign_are_refused():
    from tensorgrad_b200.ops import paged_attention

    q, pool = _t((1, 2, 8)), _pool()
    with pytest.raises(IndexError, match="page ids"):
        paged_attention(q, pool, pool, np.array([[2**64 - 1]], np.uint64), np.array([1]))
    with pytest.raises(IndexError, match="lengths must be in"):
        paged_attention(q, pool, pool, np.array([[0]]), np.array([2**64 - 1], np.uint64))


def test_a_single_number_is_no_vector_of_lengths():
    from tensorgrad_b200.ops import paged_attention

    q, pool = _t((1, 2, 8)), _pool()
    with pytest.raises(ValueError, match="expected lengths"):
        paged_attention(q, pool, pool, np.array([[0]]), np.array(1, np.uint8))
