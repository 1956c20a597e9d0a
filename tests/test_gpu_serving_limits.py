"""The serving operators at the edge of what they take: errors that name their cause."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_a_bad_device_target_names_its_operators():
    import tensorgrad_b200 as tg

    x = tg.Tensor(np.zeros((3, 4), np.float32))
    with pytest.raises(IndexError, match="class target out of range.*token_log_probs"):
        tg.token_log_probs(x, tg.Tensor(np.array([0, 4, 1]))).log_probs.numpy()
    with pytest.raises(IndexError, match="class target out of range.*cross_entropy"):
        tg.cross_entropy(x, tg.Tensor(np.array([0, -1, 1]))).numpy()
