"""``token_log_probs`` keeps a low class's digits: its probability in the gradient, and what many
equal low classes add to the sums, are as exact as the type's exponential.

Tolerances. The largest logit of every row is 0, so x - m is exact, and the other logits lie so
far below it that s - 1 is below 2^-7. With h half a step of the type, the exponential is off by
at most 4 h (two steps). A class's probability e^(x - m) / s rounds in 1 + (s - 1), the reciprocal
and the product, and s itself brings less than h: 8 h. The entropy's bracket log p + H rounds twice
more, in a difference and a product, and the part of it that is not x - m is at most 2^-7 of it and
off by less than 2^8 h relative to itself: 12 h. The sum over n equal classes of a lane rounds at
most n times, each of up to 11 joins twice; log1p, the quotient and a last addition of two
positive terms add at most 12 h.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("classes", [65, 1000, 1501, 5000, 50304])
def test_gradient_of_low_classes(classes, dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(classes)
    rows = 4
    # Multiples of 2^-12 in [-80, -16]: 50304 e^-16 < 2^-7.
    z = -16 - rng.integers(0, 64 << 12, (rows, classes)) / 4096.0
    t = rng.integers(0, classes, rows)
    r = np.arange(rows)
    z[r, t] = 0
    zl = z.astype(np.longdouble)
    e = np.exp(zl)
    e[r, t] = 0
    rest = e.sum(-1, keepdims=True)
    p = e / (1 + rest)
    ent = np.log1p(rest) - (e * zl).sum(-1, keepdims=True) / (1 + rest)
    h = float(np.finfo(dtype).eps) / 2
    for name, want, steps in (("log_probs", -p, 8),
                              ("entropy", -p * (zl - np.log1p(rest) + ent), 12)):
        x = tg.Tensor(z.astype(dtype), requires_grad=True)
        getattr(tg.token_log_probs(x, t), name).sum().backward()
        err = np.abs(x.grad.numpy() - want)
        err[r, t] = 0
        assert np.all(err <= steps * h * np.abs(want)), (name, float((err / (h * np.abs(want) + 1e-300)).max()))


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("classes", [1000, 1025, 1500, 5000])
def test_sums_over_equal_low_classes(classes, dtype):
    import tensorgrad_b200 as tg

    rows = 96
    low = -64 - np.arange(rows) * (977 / 4096)  # exact in both types, down to -86.7
    x = np.repeat(low[:, None], classes, 1)
    t = np.arange(rows) * 7 % classes
    x[np.arange(rows), t] = 0
    got = tg.token_log_probs(tg.Tensor(x.astype(dtype)), t)
    zl = low.astype(np.longdouble)
    rest = (classes - 1) * np.exp(zl)
    lanes = 32 if classes <= 1024 else 256
    h = float(np.finfo(dtype).eps) / 2
    tol = (4 + -(-classes // lanes) + 2 * 11 + 12) * h
    for have, want in ((got.log_probs.numpy(), -np.log1p(rest)),
                       (got.entropy.numpy(), np.log1p(rest) - rest * zl / (1 + rest))):
        rel = np.abs(have - want) / np.abs(want)
        assert np.all(rel <= tol), float(rel.max() / h)


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("classes", [1000, 1500, 50304])
def test_few_open_classes_side_by_side(classes, dtype):
    """Open classes that one lane reads together with the maximum, all others closed."""
    import tensorgrad_b200 as tg

    rows = 96
    low = -64 - np.arange(rows) * (977 / 4096)
    x = np.full((rows, classes), -np.inf)
    x[:, 400:404] = low[:, None]  # a 16-byte group in float, two of them in double
    t = 400 + np.arange(rows) % 4
    x[np.arange(rows), t] = 0
    got = tg.token_log_probs(tg.Tensor(x.astype(dtype)), t)
    zl = low.astype(np.longdouble)
    rest = 3 * np.exp(zl)
    h = float(np.finfo(dtype).eps) / 2
    tol = (4 + 4 + 2 * 11 + 12) * h
    for have, want in ((got.log_probs.numpy(), -np.log1p(rest)),
                       (got.entropy.numpy(), np.log1p(rest) - rest * zl / (1 + rest))):
        rel = np.abs(have - want) / np.abs(want)
        assert np.all(rel <= tol), float(rel.max() / h)
