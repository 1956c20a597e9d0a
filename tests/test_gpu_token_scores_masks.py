"""``token_log_probs`` on rows whose closed classes hold a very low finite value instead of
``-inf``: the scores are those of the open classes, and each gradient is finite on its own.

Tolerances. A closed class adds an exact 0. A term of the sums over the K open ones passes at
most K additions in its lane and 11 joins, and as many scalings: each of these 2 (K + 11) steps
rounds once, a scaling also brings its factor's error, at most 4 h + 3.4 h for each unit by which
the maximum moves (h half a step of the type; the float exponential is off by (4 + 2.4 |x|) h, its
argument rounds by |x| h), and all moves together are no longer than the spread Z of the open
logits. The term's own exponential counts the same. So the sums are off by at most
``delta = (2 (K + 11) + 4 (K + 12) + 2 * 3.4 Z) h``, relative to the sum of their terms'
magnitudes.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

OPEN = 8


def _rows(rows, classes, dtype, fill, layout, seed):
    """Logits with OPEN open classes a row, scattered, at the front or at the back, the last row
    closed but for one class."""
    rng = np.random.default_rng(seed)
    x = np.full((rows, classes), fill, dtype=dtype)
    open_ = np.empty((rows, OPEN), np.int64)
    for r in range(rows):
        if layout == "scattered":
            open_[r] = np.sort(rng.choice(classes, OPEN, replace=False))
        else:
            start = 0 if layout == "front" else classes - OPEN
            open_[r] = start + np.arange(OPEN)
    vals = (3 * rng.standard_normal((rows, OPEN))).astype(dtype)
    np.put_along_axis(x, open_, vals, -1)
    return x, open_, vals, open_[np.arange(rows), rng.integers(0, OPEN, rows)]


def _reference(vals):
    v = vals.astype(np.longdouble)
    z = v - v.max(-1, keepdims=True)
    lp = z - np.log(np.exp(z).sum(-1, keepdims=True))
    return lp, -(np.exp(lp) * lp).sum(-1), z


def _delta(z, dtype):
    h = float(np.finfo(dtype).eps) / 2
    spread = np.abs(z).max(-1).astype(np.float64)
    return (2 * (OPEN + 11) + 4 * (OPEN + 12) + 2 * 3.4 * spread) * h, h


FILLS = {"lowest": lambda t: np.finfo(t).min, "1e38": lambda t: -1e38, "-inf": lambda t: -np.inf}


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("fill", list(FILLS))
@pytest.mark.parametrize("layout", ["scattered", "front", "back"])
@pytest.mark.parametrize("rows,classes", [(3, 40), (5, 1000), (4, 1500), (300, 1501), (3, 5000),
                                          (320, 5003), (2, 50304)])
def test_closed_by_low_values(rows, classes, layout, fill, dtype):
    import tensorgrad_b200 as tg

    x, open_, vals, t = _rows(rows, classes, dtype, FILLS[fill](dtype), layout, classes)
    lp, ent, z = _reference(vals)
    delta, h = _delta(z, dtype)
    at = (open_ == t[:, None]).argmax(-1)
    r = np.arange(rows)
    given = lp[r, at]

    def leaf():
        leaf_ = tg.Tensor(x, requires_grad=True)
        return leaf_, tg.token_log_probs(leaf_, t, top_k=OPEN)

    tx, got = leaf()
    # log s is off by delta; m and the differences round by h of their sizes.
    spread = np.abs(z).max(-1).astype(np.float64)
    tol = delta + 4 * h * (spread + np.abs(given) + np.log(OPEN))
    assert np.all(np.abs(got.log_probs.numpy() - given) <= tol)
    order = np.argsort(-vals, axis=-1, kind="stable")
    np.testing.assert_array_equal(got.top_ids.numpy(), np.take_along_axis(open_, order, -1))
    # log s, and the weighted sum sum p |z| <= Z, each to delta.
    tol_ent = (delta + 4 * h) * (1 + spread) + 4 * h * np.log(OPEN)
    assert np.all(np.abs(got.entropy.numpy() - ent) <= tol_ent)

    # Each gradient alone; the closed classes get none. p is off by delta, its exponential and
    # three roundings; the entropy's bracket by tol_ent and its own roundings.
    p = np.exp(lp)
    p_tol = p * (delta + 8 * h)[:, None]
    got.log_probs.sum().backward()
    g = tx.grad.numpy()
    want = -p.copy()
    want[r, at] += 1
    assert np.all(np.abs(np.take_along_axis(g, open_, -1) - want) <= p_tol + 4 * h)
    np.put_along_axis(g, open_, 0, -1)
    assert not g.any()

    tx, got = leaf()
    got.entropy.sum().backward()
    g = tx.grad.numpy()
    want = -p * (lp + ent[:, None])
    bracket = 2 * tol_ent[:, None] + 4 * h * (np.abs(z) + 1).astype(np.float64)
    assert np.all(np.abs(np.take_along_axis(g, open_, -1) - want)
                  <= p_tol * np.abs(lp + ent[:, None]) + p * bracket + 1e-300)
    np.put_along_axis(g, open_, 0, -1)
    assert not g.any()

    tx, got = leaf()
    got.top_log_probs.sum().backward()
    g = tx.grad.numpy()
    want = 1 - OPEN * p
    assert np.all(np.abs(np.take_along_axis(g, open_, -1) - want) <= OPEN * p_tol + 4 * OPEN * h)
    np.put_along_axis(g, open_, 0, -1)
    assert not g.any()


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("classes", [40, 1500, 50304])
def test_low_values_throughout_and_beside_what_is_not_finite(classes, dtype):
    """All classes at the lowest value share the probability; a lowest value beside an infinity
    or a NaN hides neither."""
    import tensorgrad_b200 as tg

    low, high = np.finfo(dtype).min, np.finfo(dtype).max
    x = np.full((5, classes), low, dtype=dtype)
    x[1, classes // 2] = high  # further apart than the type reaches
    x[2, classes // 2] = np.nan
    x[3, classes // 3] = np.inf
    x[4, ::2] = -np.inf
    t = np.array([0, classes // 2, 0, 0, 1])
    got = tg.token_log_probs(tg.Tensor(x), t, top_k=1)
    lp, ent = got.log_probs.numpy(), got.entropy.numpy()
    h = float(np.finfo(dtype).eps) / 2
    # Sums of ones are exact; log, and the last difference, round to 2 h of log(classes) each.
    assert abs(lp[0] + np.log(classes)) <= 4 * h * np.log(classes)
    assert abs(ent[0] - np.log(classes)) <= 4 * h * np.log(classes)
    assert lp[1] == 0 and ent[1] == 0
    assert np.isnan(lp[2]) and np.isnan(ent[2]) and np.isnan(lp[3]) and np.isnan(ent[3])
    half = classes // 2
    assert abs(lp[4] + np.log(half)) <= 4 * h * np.log(half)
    assert abs(ent[4] - np.log(half)) <= 4 * h * np.log(half)
    np.testing.assert_array_equal(got.top_ids.numpy()[[0, 1, 3, 4], 0],
                                  [0, classes // 2, classes // 3, 1])
