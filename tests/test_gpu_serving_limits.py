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


def test_int8_linear_float64_beyond_four_million_rows():
    """More rows than a launch grid's second axis has tiles of 64. The integers of a row of two
    values are +-127 and the nearest integer of a quotient, so the product is restated exactly."""
    import tensorgrad_b200 as tg

    rows, inner, outer = 64 * 65536 + 1, 2, 3
    rng = np.random.default_rng(0)
    x = rng.standard_normal((rows, inner))
    w = rng.integers(-127, 128, (outer, inner)).astype(np.int8)
    scale = rng.uniform(0.5, 2, outer)
    got = tg.int8_linear(tg.Tensor(x), tg.Int8Weight(w, scale)).numpy()
    sx = np.abs(x).max(-1) * (1.0 / 127)
    q = np.rint(x / sx[:, None])
    want = (q @ w.T.astype(np.float64)) * (sx[:, None] * scale)
    # Two roundings of the product on either side.
    assert np.all(np.abs(got - want) <= 4 * np.finfo(np.float64).eps / 2 * np.abs(want))
