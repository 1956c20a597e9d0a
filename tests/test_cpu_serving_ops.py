"""Refusals and host logic of the serving operators, without a GPU: the wrappers check their
arguments before they touch device memory, the C entry points before they launch."""

from __future__ import annotations

import numpy as np
import pytest


class _Meta:
    """Stands in for device data: the checks read shapes and types only."""

    def __init__(self, shape, dtype=np.float32):
        self.shape = tuple(shape)
        self.ndim = len(self.shape)
        self.dtype = np.dtype(dtype)
        self.size = int(np.prod(self.shape))


def _t(shape, dtype=np.float32):
    from tensorgrad_b200.tensor import Tensor

    return Tensor._wrap(_Meta(shape, dtype))


def test_token_log_probs_refuses_bad_arguments():
    from tensorgrad_b200.ops import token_log_probs

    with pytest.raises(ValueError, match="class axis"):
        token_log_probs(_t(()), 0)
    with pytest.raises(ValueError, match="class axis"):
        token_log_probs(_t((2, 0)), np.zeros(2, np.int64))
    for k in (-1, 8, 129):
        with pytest.raises(ValueError, match="top_k must be in"):
            token_log_probs(_t((2, 7)), np.zeros(2, np.int64), top_k=k)
    with pytest.raises(ValueError, match=r"top_k must be in \[0, 128\]"):
        token_log_probs(_t((2, 700)), np.zeros(2, np.int64), top_k=129)
    with pytest.raises(TypeError, match="integers"):
        token_log_probs(_t((2, 7)), np.zeros(2))
    with pytest.raises(ValueError, match="incompatible"):
        token_log_probs(_t((2, 7)), np.zeros(3, np.int64))
    for bad in (7, -1):
        with pytest.raises(IndexError, match="7 classes"):
            token_log_probs(_t((2, 7)), np.array([0, bad]))


def test_token_log_probs_entry_points_refuse_bad_sizes():
    from tensorgrad_b200._lib import last_error, lib

    def forward(rows, classes, top_k, dtype=0):
        return lib.tg_token_log_probs_forward(dtype, *[None] * 7, rows, classes, top_k, -100,
                                              None, None, None)

    assert forward(2, 0, 0) == 1
    assert forward(-1, 5, 0) == 1
    assert forward(2, 1 << 31, 0) == 1
    assert forward(2, 5, 6) == 1 and "top_k 6" in last_error()
    assert forward(2, 500, 129) == 1
    assert forward(2, 500, 4) == 1 and "no room" in last_error()
    assert forward(0, 500, 0) == 0
    assert lib.tg_token_log_probs_backward(0, *[None] * 9, 2, 0, 0, -100, None) == 1
