"""Linear layers in 8-bit integers: the integers and scales exactly as the input's type rounds
them, the outputs from exact integer sums.

Tolerance: the integer sum is exact; its conversion, the product of the two scales, their
product and the bias round once each, so an output is off by at most 3 h |sum s s'| (1 + h)^3
+ h |y| with h half a step of the type: 4 h (|sum s s'| + |y|) bounds it.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[np.float32, np.float64], ids=["fp32", "fp64"])
def dtype(request):
    return request.param


def _quantized(x):
    """(integers, scales) as the type of ``x`` rounds them."""
    scale = np.abs(x).max(-1) * (x.dtype.type(1) / x.dtype.type(127))
    safe = np.where(scale > 0, scale, 1)[..., None].astype(x.dtype)
    q = np.clip(np.rint(x / safe), -127, 127) * (scale > 0)[..., None]
    return q.astype(np.int8), scale


def _check(y, x, q, scale, bias):
    a, s = _quantized(x)
    total = a.astype(np.float64) @ q.astype(np.float64).T  # integers below 2^53: exact
    prod = total.astype(np.longdouble) * s[:, None].astype(np.longdouble) * scale.astype(np.longdouble)
    ref = prod if bias is None else prod + bias
    h = np.finfo(x.dtype).eps / 2
    err = np.abs(y - ref) - 4 * h * (np.abs(prod) + np.abs(ref))
    assert y.dtype == x.dtype
    assert err.max() <= 1e-300, float(err.max())


SHAPES = [(1, 1, 1), (1, 768, 2304), (7, 16, 1), (2, 17, 5), (8, 4096, 300), (9, 100, 70),
          (16, 768, 1000), (33, 1001, 77), (128, 64, 256), (129, 130, 65), (300, 4096, 513),
          (1, 8192, 40), (2000, 256, 640), (1025, 48, 2052), (64, 2000, 129), (257, 1024, 4096),
          (1, 48128, 5), (1, 49000, 3), (2, 24064, 4), (5, 6016, 9), (8, 6100, 7), (16, 4096, 4100),
          (2100, 130, 4500), (2049, 2100, 4100), (600, 3000, 8195)]


@pytest.mark.parametrize("rows,inner,outer", SHAPES)
def test_linear_matches_integer_sums(rows, inner, outer, dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(rows + inner + outer)
    x = rng.standard_normal((rows, inner)).astype(dtype)
    x[:, rng.integers(inner, size=max(1, inner // 50))] *= 20
    w = rng.standard_normal((outer, inner)).astype(dtype)
    bias = rng.standard_normal(outer).astype(dtype) if rows % 2 else None
    weight = tg.Int8Weight.quantize(tg.Tensor(w))
    q, scale = _quantized(w)
    np.testing.assert_array_equal(weight.q.numpy()[:, :inner], q)
    assert not weight.q.numpy()[:, inner:].any()
    np.testing.assert_array_equal(weight.scale.numpy(), scale)
    y = tg.int8_linear(tg.Tensor(x), weight, None if bias is None else tg.Tensor(bias)).numpy()
    _check(y, x, q, scale, bias)
    xq, xs = tg.quantize_int8(tg.Tensor(x))
    a, s = _quantized(x)
    assert xq.dtype == np.int8
    np.testing.assert_array_equal(xq.numpy(), a)
    np.testing.assert_array_equal(xs.numpy(), s)


@pytest.mark.parametrize("rows", [1, 5, 200])
def test_largest_sums_stay_exact(rows, dtype):
    import tensorgrad_b200 as tg

    inner = 131072
    x = np.ones((rows, inner), dtype)
    x[:, 1::2] = -1
    q = np.full((3, inner), 127, np.int8)
    q[:, 1::2] = -128
    q[2] = -128
    weight = tg.Int8Weight(q, np.array([1, 0.5, 2], dtype))
    _check(tg.int8_linear(tg.Tensor(x), weight).numpy(), x, q, np.array([1, 0.5, 2], dtype), None)


def test_halves_zeros_and_tiny_rows(dtype):
    import tensorgrad_b200 as tg

    tiny = np.finfo(dtype).smallest_subnormal
    x = np.array([[127, 0.5, 1.5, -2.5, 0, 126.5], [0, 0, 0, 0, 0, 0],
                  [tiny, -tiny, 0, tiny, 0, 0],
                  [200 * tiny, 3 * tiny, -tiny, 0, 0, 0]], dtype)
    q, s = tg.quantize_int8(tg.Tensor(x))
    a, scale = _quantized(x)
    np.testing.assert_array_equal(q.numpy(), a)
    np.testing.assert_array_equal(s.numpy(), scale)
    np.testing.assert_array_equal(q.numpy()[0], [127, 0, 2, -2, 0, 126])
    assert not q.numpy()[1].any() and s.numpy()[1] == 0


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_rows_that_are_not_finite_spoil_themselves_only(rows, dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, 80)).astype(dtype)
    weight = tg.Int8Weight.quantize(tg.Tensor(rng.standard_normal((70, 80)).astype(dtype)))
    clean = tg.int8_linear(tg.Tensor(x), weight).numpy()
    x[0, 79], x[rows - 1, 3] = np.nan, -np.inf
    y = tg.int8_linear(tg.Tensor(x), weight).numpy()
    assert np.all(np.isnan(y[[0, rows - 1]]))
    np.testing.assert_array_equal(y[1:rows - 1], clean[1:rows - 1])


def test_weights_in_other_layouts_and_types():
    import tensorgrad_b200 as tg
    from tensorgrad_b200 import device

    rng = np.random.default_rng(6)
    x = rng.standard_normal((5, 4, 19)).astype(np.float32)
    q = rng.integers(-128, 128, (33, 19)).astype(np.int8)
    scale = rng.random(33).astype(np.float32)
    want = tg.int8_linear(tg.Tensor(x), tg.Int8Weight(q, scale)).numpy()
    _check(want.reshape(20, 33), x.reshape(20, 19), q, scale, None)
    junk = np.full((33, 32), 99, np.int8)  # what lies behind in_features does not count
    junk[:, :19] = q
    dev = device.from_numpy(junk)
    assert tg.Int8Weight(dev, scale, 19).q is dev
    flat = device.from_numpy(np.concatenate([[0], junk.reshape(-1)]).astype(np.int8))
    for other in (dev, device.from_numpy(q), flat.flat_view(1, junk.size, junk.shape)):
        got = tg.int8_linear(tg.Tensor(x), tg.Int8Weight(other, scale.astype(np.float64), 19))
        np.testing.assert_array_equal(got.numpy(), want)
    # Inputs and outputs of any alignment.
    off = device.from_numpy(np.concatenate([[0], x.reshape(-1)]).astype(np.float32))
    view = tg.Tensor._wrap(off.flat_view(1, x.size, x.shape))
    np.testing.assert_array_equal(tg.int8_linear(view, tg.Int8Weight(q, scale)).numpy(), want)
    empty = tg.int8_linear(tg.Tensor(np.zeros((0, 19), np.float32)), tg.Int8Weight(q, scale))
    assert empty.shape == (0, 33)


def test_quantized_model_serves_and_saves():
    import tensorgrad_b200 as tg

    def model():
        tg.set_default_dtype(np.float64)
        tg.manual_seed(5)
        m = tg.nn.GPT(tg.nn.GPTConfig(vocab_size=61, block_size=32, n_layer=2, n_head=4, n_embd=48))
        tg.set_default_dtype(np.float32)
        return m.quantize_int8(head=True)

    m = model()
    linear = [x for _, x in m.named_modules() if isinstance(x, tg.nn.Linear)]
    assert not linear and not any(p.requires_grad for p in m.parameters())
    assert sum(isinstance(x, tg.nn.Int8Linear) for _, x in m.named_modules()) == 9
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 61, n) for n in (4, 9)]
    # In float64 the paths differ by rounding far below a step of the integers, so the pages,
    # the contiguous cache and the whole forward agree.
    for p, (s,) in zip(prompts, m.generate_batch(prompts, 6, top_k=1, page_size=4), strict=True):
        np.testing.assert_array_equal(s.ids, m.generate(p[None], 6, top_k=1)[0])
        logits = m(s.ids[None]).numpy()[0]
        lp = logits - np.log(np.exp(logits).sum(-1, keepdims=True))
        at = np.arange(len(p) - 1, len(s.ids) - 1)
        np.testing.assert_allclose(s.log_probs, lp[at, s.ids[at + 1]], rtol=0, atol=1e-10)
    state = m.state_dict()
    assert state["blocks.0.attn.qkv.weight"].dtype == np.int8
    other = model()
    before = other(prompts[0][None]).numpy()
    other.load_state_dict({k: np.zeros_like(v) for k, v in state.items()})
    assert not other(prompts[0][None]).numpy().any()
    other.load_state_dict(state)
    np.testing.assert_array_equal(other(prompts[0][None]).numpy(), before)


def test_int8_layer_is_the_operator():
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(2)
    layer = tg.nn.Linear(40, 24)
    small = tg.nn.Int8Linear(layer)
    x = rng.standard_normal((3, 40)).astype(np.float32)
    _check(small(tg.Tensor(x)).numpy(), x, *_quantized(layer.weight.numpy()), layer.bias.numpy())
    with pytest.raises(ValueError, match="inference"):
        small(tg.Tensor(x, requires_grad=True))
    with tg.no_grad():
        small(tg.Tensor(x, requires_grad=True))


@pytest.mark.parametrize("rows,inner,outer", [(300, 256, 700), (2049, 2100, 4100)])
def test_wait_that_runs_out_reports_and_recovers(rows, inner, outer):
    """The bounded waits of the tensor-core product (one CTA to a tile, and a pair): with no
    load issued and a budget of about a millisecond the first wait gives up, the kernel drains
    with nothing in flight, and the next synchronisation raises; afterwards the same call is
    right again."""
    import tensorgrad_b200 as tg
    from tensorgrad_b200 import device
    from tensorgrad_b200._lib import check, lib

    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    w = rng.standard_normal((outer, inner)).astype(np.float32)
    weight, tx = tg.Int8Weight.quantize(tg.Tensor(w)), tg.Tensor(x)
    device.synchronize()
    check(lib.tg_int8_set_wait_test(2_000_000, 1))
    try:
        y = tg.int8_linear(tx, weight)
        with pytest.raises(RuntimeError, match="8-bit integer linear: a bounded device-side wait"):
            device.synchronize()
        del y
    finally:
        check(lib.tg_int8_set_wait_test(0, 0))
    device.synchronize()
    _check(tg.int8_linear(tx, weight).numpy(), x, *_quantized(w), None)
