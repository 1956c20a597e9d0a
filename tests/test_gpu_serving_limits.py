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


@pytest.mark.parametrize("size", [0, -4])
def test_generate_batch_refuses_a_page_size_below_one(size):
    import tensorgrad_b200 as tg

    model = tg.nn.GPT(tg.nn.GPTConfig(vocab_size=11, block_size=16, n_layer=1, n_head=1,
                                      n_embd=8))
    for new in (0, 3):
        with pytest.raises(ValueError, match=f"page_size must be positive, got {size}"):
            model.generate_batch([np.array([1, 2])], new, page_size=size)
    assert model.training
