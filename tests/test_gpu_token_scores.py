"""``token_log_probs`` against its definition in extended precision, its order of
alternatives, its gradients against the formula and against differences, and its refusals.

Tolerances. A row's statistics are sums of positive terms in which every value passes through
a fixed number of roundings: with n values to a thread, each step of the running sum rounds
at most 4 times (two scalings, exponential, addition; the exponential itself is off by at most
4 half steps), and 16 joins follow, so the relative error of s is at most
``delta = 12 (n + 16) h`` with h half a step of the type; log s is then off by delta
absolutely, and the entropy's weighted sum by delta times (1 + sum p |x - m|). Each value
also rounds once or twice itself, relative to its size: 8 h (|x - m| + |log s| + H).
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

THREADS = 128  # the fewest threads that share a row


def _half(dtype) -> float:
    return float(np.finfo(dtype).eps) / 2


def _inputs(rows, classes, dtype, seed, closed=True, scale=3.0):
    rng = np.random.default_rng(seed)
    x = (scale * rng.standard_normal((rows, classes))).astype(dtype)
    shut = classes // 50 if closed else 0
    if shut:
        x[:, classes - shut:] = -np.inf
    t = rng.integers(0, classes - shut, rows)
    t[rng.random(rows) < 0.2] = -100
    return x, t


def _definition(x, t, top_k, ignore=-100):
    """(log_probs, entropy, top log probs, top ids, p, log p) in extended precision."""
    x = x.astype(np.longdouble)
    m = x.max(-1, keepdims=True)
    e = np.exp(x - m)
    lp = x - m - np.log(e.sum(-1, keepdims=True))
    p = np.exp(lp)
    ent = -(p * np.where(p > 0, lp, 0)).sum(-1)
    rows = np.arange(len(t))
    given = np.where(t == ignore, 0, lp[rows, np.where(t == ignore, 0, t)])
    ids = np.argsort(-x, axis=-1, kind="stable")[:, :top_k]
    return given, ent, np.take_along_axis(lp, ids, -1), ids, p, lp


def _bounds(x, dtype):
    """Per row: the absolute error that log s and the entropy may have, and the spread
    sum p |x - m| they scale with."""
    h = _half(dtype)
    xl = x.astype(np.longdouble)
    z = xl - xl.max(-1, keepdims=True)
    e = np.exp(z)
    spread = (e * np.where(e > 0, -z, 0)).sum(-1) / e.sum(-1)
    ls = np.abs(np.log(e.sum(-1)))
    delta = 12 * (-(-x.shape[-1] // THREADS) + 16) * h
    return (delta * (1 + spread) + 8 * h * (1 + spread + ls)).astype(np.float64), spread, ls


SHAPES = [(1, 1, 1), (1, 17, 5), (3, 65, 65), (5, 1000, 20), (2, 4099, 128), (9, 50304, 5),
          (300, 257, 3), (1, 131072, 20), (700, 1024, 0), (4, 300, 128), (77, 1025, 9),
          (9, 129, 128), (2, 128, 128)]


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("rows,classes,top_k", SHAPES)
def test_scores_match_definition(rows, classes, top_k, dtype):
    import tensorgrad_b200 as tg

    x, t = _inputs(rows, classes, dtype, rows + classes)
    got = tg.token_log_probs(tg.Tensor(x), t, top_k=top_k)
    given, ent, top, ids, _, _ = _definition(x, t, top_k)
    tol, _, _ = _bounds(x, dtype)
    h = _half(dtype)
    assert got.log_probs.shape == (rows,) and got.log_probs.dtype == dtype
    assert np.all(np.abs(got.log_probs.numpy() - given) <= tol + 4 * h * np.abs(given))
    assert np.all(got.log_probs.numpy()[t == -100] == 0)
    assert np.all(np.abs(got.entropy.numpy() - ent) <= 2 * tol + 4 * h * np.abs(ent))
    if not top_k:
        assert got.top_log_probs is None and got.top_ids is None
        return
    np.testing.assert_array_equal(got.top_ids.numpy(), ids)
    top_got = got.top_log_probs.numpy()
    open_ = np.isfinite(top.astype(np.float64))
    np.testing.assert_array_equal(np.isfinite(top_got), open_)
    err = np.where(open_, np.abs(top_got - np.where(open_, top, 0)), 0)
    assert np.all(err <= tol[:, None] + 4 * h * np.where(open_, np.abs(top), 0))


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("rows,classes,top_k", [(1, 1, 1), (3, 65, 7), (5, 4099, 20),
                                                (300, 257, 0), (2, 50304, 128), (19, 1025, 3),
                                                (500, 1024, 2)])
def test_gradient_matches_formula(rows, classes, top_k, dtype):
    import tensorgrad_b200 as tg

    x, t = _inputs(rows, classes, dtype, 7 * rows + classes)
    rng = np.random.default_rng(3)
    gl, ge = rng.standard_normal((2, rows)).astype(dtype)
    gt = rng.standard_normal((rows, top_k)).astype(dtype)
    tx = tg.Tensor(x, requires_grad=True)
    got = tg.token_log_probs(tx, t, top_k=top_k)
    outs, grads = [got.log_probs, got.entropy], [gl, ge]
    if top_k:
        outs.append(got.top_log_probs)
        grads.append(gt)
    tg.autograd.backward(outs, grads)
    _, ent, _, ids, p, lp = _definition(x, t, top_k)
    kept = t != -100
    pull = (gl * kept).astype(np.longdouble)
    all_ = pull + gt.astype(np.longdouble).sum(-1)
    slp = np.where(p > 0, lp, 0)
    ref = -p * (all_[:, None] + ge[:, None] * (slp + ent[:, None]))
    r = np.arange(rows)
    ref[r[kept], t[kept]] += pull[kept]
    for k in range(top_k):
        ref[r, ids[:, k]] += gt[:, k]
    tol, spread, ls = _bounds(x, dtype)
    h = _half(dtype)
    # p carries the error of s and of its own exponential; the bracket that of the entropy and
    # of the sum over the alternatives; the gradients added at single classes round once each.
    size = (np.abs(pull) + np.abs(gt).sum(-1))[:, None] + np.abs(ge)[:, None] * (
        np.abs(slp) + np.abs(ent)[:, None] + 1)
    added = np.abs(ref) + p * size
    bound = (p * size * (2 * tol + (24 + 2 * top_k) * h)[:, None]
             + p * np.abs(ge)[:, None] * 2 * tol[:, None] + 8 * h * added)
    err = np.abs(tx.grad.numpy() - ref)
    assert np.all(err <= bound + 1e-300), float((err - bound).max())


def test_ties_go_to_the_lowest_class():
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(0)
    for rows, classes, top_k in [(3, 5000, 128), (2, 70001, 64), (200, 300, 100), (1, 131, 128),
                                 (400, 20000, 30), (5, 1100, 20)]:
        for levels in (1, 3, 40):
            x = rng.integers(0, levels, (rows, classes)).astype(np.float32)
            x[rng.random(x.shape) < 0.1] *= -0.0  # both zeros count as equal
            got = tg.token_log_probs(tg.Tensor(x), np.zeros(rows, np.int64), top_k=top_k)
            ids = np.argsort(-x, axis=-1, kind="stable")[:, :top_k]
            np.testing.assert_array_equal(got.top_ids.numpy(), ids)


@pytest.mark.parametrize("classes", [40, 5000])
def test_rows_without_a_distribution(classes):
    import tensorgrad_b200 as tg

    x = np.random.default_rng(1).standard_normal((5, classes)).astype(np.float32)
    x[0] = -np.inf
    x[1, 3] = np.nan
    x[2, 7] = np.inf
    x[3, 1:] = -np.inf  # one class left: certain
    tx = tg.Tensor(x, requires_grad=True)
    got = tg.token_log_probs(tx, np.zeros(5, np.int64), top_k=20)
    lp, ent, ids = got.log_probs.numpy(), got.entropy.numpy(), got.top_ids.numpy()
    assert np.all(np.isnan(lp[:3])) and np.all(np.isnan(ent[:3]))
    assert lp[3] == 0 and ent[3] == 0 and np.isfinite(lp[4])
    for row in ids:
        assert len(set(row.tolist())) == 20 and row.min() >= 0 and row.max() < classes
    np.testing.assert_array_equal(ids[0], np.arange(20))
    assert ids[2, 0] == 7 and 3 not in ids[1]
    np.testing.assert_array_equal(got.top_log_probs.numpy()[3], [0] + [-np.inf] * 19)
    tg.autograd.backward([got.log_probs, got.entropy], [np.ones(5), np.ones(5)])
    g = tx.grad.numpy()
    assert np.all(g[3] == 0) and np.all(np.isfinite(g[4])) and np.all(np.isnan(g[0]))


def test_batched_logits_device_targets_and_unaligned_views():
    import tensorgrad_b200 as tg
    from tensorgrad_b200 import device

    x, t = _inputs(6, 4096, np.float32, 5)
    flat = tg.token_log_probs(tg.Tensor(x), t, top_k=3)
    cube = tg.token_log_probs(tg.Tensor(x.reshape(2, 3, 4096)), tg.Tensor(t.reshape(2, 3)),
                              top_k=3)
    assert cube.entropy.shape == (2, 3) and cube.top_ids.shape == (2, 3, 3)
    for a, b in zip(flat, cube, strict=True):
        np.testing.assert_array_equal(a.numpy().reshape(-1), b.numpy().reshape(-1))
    buf = device.from_numpy(np.concatenate([[0], x.reshape(-1)]).astype(np.float32))
    shifted = tg.Tensor._wrap(buf.flat_view(1, x.size, x.shape))
    off = tg.token_log_probs(shifted, t, top_k=3)
    tol, _, _ = _bounds(x, np.float32)
    assert np.all(np.abs(off.entropy.numpy() - flat.entropy.numpy()) <= 4 * tol)
    np.testing.assert_array_equal(off.top_ids.numpy(), flat.top_ids.numpy())
    empty = tg.token_log_probs(tg.Tensor(np.zeros((0, 5), np.float32)), np.zeros(0, np.int64),
                               top_k=2)
    assert empty.log_probs.shape == (0,) and empty.top_ids.shape == (0, 2)


def test_device_target_out_of_range_raises_at_the_next_synchronisation():
    import tensorgrad_b200 as tg

    got = tg.token_log_probs(tg.Tensor(np.zeros((3, 4), np.float32)), tg.Tensor(np.array([0, 4, 1])))
    with pytest.raises(IndexError):
        got.log_probs.numpy()
    again = tg.token_log_probs(tg.Tensor(np.zeros((3, 4), np.float32)), tg.Tensor(np.array([0, -100, 1])))
    np.testing.assert_allclose(again.log_probs.numpy(), [-np.log(4), 0, -np.log(4)], rtol=1e-6)


def test_gradients_against_differences():
    import tensorgrad_b200 as tg
    from tensorgrad_b200.utils import gradcheck, gradgradcheck

    rng = np.random.default_rng(9)
    x = tg.Tensor(rng.permutation(12).reshape(3, 4) * 0.3 + 0.01 * rng.random((3, 4)),
                  requires_grad=True)
    t = np.array([1, -100, 3])

    def total(a):
        got = tg.token_log_probs(a, t, top_k=2)
        return tg.concat([got.log_probs, got.entropy * 0.5, got.top_log_probs.reshape(6)])

    gradcheck(total, [x])
    gradgradcheck(total, [x])


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["fp32", "fp64"])
@pytest.mark.parametrize("classes", [7, 130, 1000, 5000, 50304])
def test_nearly_certain_tokens_keep_their_digits(classes, dtype):
    """A class 15 to 25 above the others: log p and H are of the size of e^-15, far below a step
    of 1. Relative error: every e^(x - m) is off by (4 + 2.4 |x - m|) h and one rounding of its
    argument's |x - m| h, the sum of n to a lane by 12 (n + 16) h; log1p, the quotient and the
    last addition of two positive terms by a few h. |x - m| is at most 40 here."""
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(classes)
    rows = 6
    x = rng.standard_normal((rows, classes)).astype(dtype)
    t = rng.integers(0, classes, rows)
    x[np.arange(rows), t] += np.linspace(15, 25, rows).astype(dtype)
    tx = tg.Tensor(x, requires_grad=True)
    got = tg.token_log_probs(tx, t, top_k=2)
    given, ent, top, _, p, lp = _definition(x, t, 2)
    # Extended precision has digits to spare for the definition's own 1 - p and log.
    z = x.astype(np.longdouble) - x.max(-1, keepdims=True)
    e = np.exp(z)
    e[np.arange(rows), t] = 0
    rest = e.sum(-1)
    lp_t = -np.log1p(rest)
    ent = np.log1p(rest) - (e * z).sum(-1) / (1 + rest)
    h = _half(dtype)
    rel = (12 * (-(-classes // THREADS) + 16) + 2 * (4 + 3.4 * 40) + 8) * h
    assert np.all(np.abs(got.log_probs.numpy() - lp_t) <= rel * np.abs(lp_t))
    assert np.all(np.abs(got.top_log_probs.numpy()[:, 0] - lp_t) <= rel * np.abs(lp_t))
    assert np.all(np.abs(got.entropy.numpy() - ent) <= rel * np.abs(ent))
    tg.autograd.backward([got.log_probs], [np.ones(rows)])
    want = rest / (1 + rest)  # 1 - p of the target
    g = tx.grad.numpy()[np.arange(rows), t]
    assert np.all(np.abs(g - want) <= rel * np.abs(want))


def test_each_output_alone_and_used_twice():
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(12)
    x = rng.standard_normal((4, 9))
    t = np.array([3, -100, 0, 8])
    g = [rng.standard_normal(4), rng.standard_normal(4), rng.standard_normal((4, 3))]

    def grads(wanted, times=1):
        tx = tg.Tensor(x, requires_grad=True)
        got = tg.token_log_probs(tx, t, top_k=3)
        outs = [got.log_probs, got.entropy, got.top_log_probs]
        total = None
        for i in wanted:
            for _ in range(times):
                term = (outs[i] * tg.Tensor(g[i] / times)).sum()
                total = term if total is None else total + term
        total.backward()
        return tx.grad.numpy()

    one = [grads([i]) for i in range(3)]
    np.testing.assert_allclose(grads([0, 1, 2]), sum(one), rtol=0, atol=1e-14)
    np.testing.assert_allclose(grads([2, 0]), one[0] + one[2], rtol=0, atol=1e-14)
    for i in range(3):
        np.testing.assert_allclose(grads([i], times=2), one[i], rtol=0, atol=1e-14)


def test_matches_cross_entropy_through_the_model_path():
    import tensorgrad_b200 as tg

    x, t = _inputs(64, 1000, np.float32, 4, closed=False)
    a, b = tg.Tensor(x, requires_grad=True), tg.Tensor(x, requires_grad=True)
    tg.cross_entropy(a, t, reduction="sum").backward()
    (-tg.token_log_probs(b, t).log_probs.sum()).backward()
    # Both are p - [j = t]: p rounds differently, by at most the bound of the statistics each.
    tol, _, _ = _bounds(x, np.float32)
    assert np.all(np.abs(a.grad.numpy() - b.grad.numpy()) <= 4 * tol[:, None])
