"""The gradient of ``token_log_probs`` is the same function with and without ``create_graph``, at
closed classes too: both are compared with the formula.

Tolerance. With h half a float64 step, sums over n classes round at most n times, and every other
value passes through fewer than 64 roundings of at most its own size; the incoming gradients add
up to at most G in a row, log p and the entropy of open classes are at most L: a class's gradient
is off by at most ``(n + 64) h G (1 + L)``.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("classes", [6, 40, 1500])
@pytest.mark.parametrize("fill", [-np.inf, np.finfo(np.float64).min], ids=["-inf", "lowest"])
def test_closed_targets_and_alternatives(classes, fill):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(classes)
    rows, top_k, opened = 5, 5, 3  # more alternatives than open classes
    x = np.full((rows, classes), fill)
    open_ = np.stack([1 + np.sort(rng.choice(classes - 1, opened, replace=False))
                      for _ in range(rows)])
    np.put_along_axis(x, open_, 2 * rng.standard_normal((rows, opened)), -1)
    closed = np.array([[c for c in range(classes) if c not in row][-1] for row in open_])
    # Targets: open, closed, closed and an alternative (class 0), none, open.
    t = np.array([open_[0, 1], closed[1], 0, -100, open_[4, 0]])
    gl, ge = rng.uniform(2, 3, (2, rows))
    gt = rng.uniform(2, 3, (rows, top_k))

    got = {}
    for mode in (False, True):
        tx = tg.Tensor(x, requires_grad=True)
        out = tg.token_log_probs(tx, t, top_k=top_k)
        ids = out.top_ids.numpy()
        each = [tg.autograd.grad([o], [tx], grad_outputs=[tg.Tensor(g)], create_graph=mode,
                                 retain_graph=True)[0].numpy()
                for o, g in ((out.log_probs, gl), (out.entropy, ge), (out.top_log_probs, gt))]
        got[mode] = each

    xl = x.astype(np.longdouble)
    z = xl - xl.max(-1, keepdims=True)
    lp = z - np.log(np.exp(z).sum(-1, keepdims=True))
    p = np.exp(lp)
    slp = np.where(p > 0, lp, 0)
    ent = -(p * slp).sum(-1, keepdims=True)
    r = np.arange(rows)
    kept = t != -100
    want_l = -p * (gl * kept)[:, None]
    want_l[r[kept], t[kept]] += gl[kept]
    want_t = -p * gt.sum(-1, keepdims=True)
    for k in range(top_k):
        want_t[r, ids[:, k]] += gt[:, k]
    want = [want_l, -p * ge[:, None] * (slp + ent), want_t]
    h = np.finfo(np.float64).eps / 2
    size = 1 + float(np.abs(slp).max()) + float(ent.max())
    for i, name in enumerate(("log_probs", "entropy", "top_log_probs")):
        for mode in (False, True):
            err = np.abs(got[mode][i] - want[i])
            assert np.all(err <= (classes + 64) * h * 3 * top_k * size), (name, mode)
