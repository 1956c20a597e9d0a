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
                                              None, None)

    assert forward(2, 0, 0) == 1
    assert forward(-1, 5, 0) == 1
    assert forward(2, 1 << 31, 0) == 1
    assert forward(2, 5, 6) == 1 and "top_k 6" in last_error()
    assert forward(2, 500, 129) == 1
    assert forward(2, 500, 4) == 1 and "no room" in last_error()
    assert forward(0, 500, 0) == 0
    assert lib.tg_token_log_probs_backward(0, *[None] * 9, 2, 0, 0, -100, None) == 1


# ---------------------------------------------------------------------- pages
def _pool(dtype=np.float32, shape=(6, 2, 4, 8)):
    return _t(shape, dtype)


def test_page_ops_refuse_bad_arguments():
    from tensorgrad_b200.ops import append_pages, copy_pages, gather_pages, paged_attention

    q, k, pool = _t((3, 4, 8)), _t((3, 2, 1, 8)), _pool()
    table, held = np.zeros((3, 2), np.int64), np.zeros(3, np.int64)
    with pytest.raises(TypeError, match="key pool must be a tensor"):
        paged_attention(q, np.zeros((6, 2, 4, 8)), pool, table, held)
    with pytest.raises(ValueError, match="expected pools"):
        paged_attention(q, _t((6, 4, 8)), _t((6, 4, 8)), table, held)
    with pytest.raises(ValueError, match="differ"):
        paged_attention(q, pool, _pool(np.float64), table, held)
    with pytest.raises(ValueError, match="differ"):
        gather_pages(pool, _pool(shape=(5, 2, 4, 8)), table, held, 3)
    for bad in (_t((3, 3, 8)), _t((3, 4, 7)), _t((4, 8)), _t((3, 0, 8))):
        with pytest.raises(ValueError, match="do not match"):
            paged_attention(bad, pool, pool, table, held)
    with pytest.raises(TypeError, match="float64 for pools of float32"):
        paged_attention(_t((3, 4, 8), np.float64), pool, pool, table, held)
    with pytest.raises(NotImplementedError, match="at most 256"):
        wide = _pool(shape=(2, 1, 1, 257))
        paged_attention(_t((3, 1, 257)), wide, wide, table, held)
    with pytest.raises(TypeError, match="pages must be integers"):
        paged_attention(q, pool, pool, table.astype(float), held)
    for pages, lengths in ((table[:2], held), (table[:, :0], held), (table, held[:2]),
                           (table[0], held)):
        with pytest.raises(ValueError, match="expected"):
            paged_attention(q, pool, pool, pages, lengths)
    for lengths in ([0, 0, 9], [0, -1, 0]):
        with pytest.raises(IndexError, match=r"lengths must be in \[0, 8\]"):
            paged_attention(q, pool, pool, table, np.array(lengths))
    for page in (6, -1):
        with pytest.raises(IndexError, match=r"page ids must be in \[0, 6\)"):
            paged_attention(q, pool, pool, np.array([[0, 9], [0, 0], [page, 0]]),
                            np.array([4, 8, 1]))
    with pytest.raises(ValueError, match="longest"):
        gather_pages(pool, pool, table, held, -1)
    with pytest.raises(IndexError, match=r"lengths must be in \[0, 7\]"):
        append_pages(k, k, pool, pool, table, np.array([0, 8, 0]))
    with pytest.raises(ValueError, match="do not match"):
        append_pages(k, _t((3, 2, 2, 8)), pool, pool, table, held)
    with pytest.raises(TypeError, match="float64"):
        append_pages(_t((3, 2, 1, 8), np.float64), k, pool, pool, table, held)
    with pytest.raises(IndexError, match="page ids"):
        copy_pages(pool, pool, [0], [6])
    with pytest.raises(ValueError, match="twice"):
        copy_pages(pool, pool, [0, 1], [2, 2])
    with pytest.raises(ValueError, match="both a source"):
        copy_pages(pool, pool, [0, 1], [1, 2])
    for src, dst in (([0, 1], [2]), (0, 1), ([[0]], [[1]])):
        with pytest.raises(ValueError, match="as many sources"):
            copy_pages(pool, pool, src, dst)
    with pytest.raises(TypeError, match="integers"):
        copy_pages(pool, pool, [0.5], [2.0])
    copy_pages(pool, pool, [], [])
    learnt = _pool()
    learnt._requires_grad = True
    with pytest.raises(ValueError, match="inference"):
        paged_attention(q, learnt, pool, table, held)


def test_page_entry_points_refuse_bad_sizes():
    from tensorgrad_b200._lib import lib

    def attend(batch=1, heads=4, kv_heads=2, width=8, pool=3, size=4, table=2, dtype=0):
        return lib.tg_paged_attention(dtype, batch, heads, kv_heads, width, None, 0, 0, None,
                                      None, pool, size, None, table, None, 1, None, None, None,
                                      None, None)

    assert attend(batch=0) == 0
    for bad in (dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(pool=0), dict(size=0),
                dict(table=0), dict(width=0), dict(batch=-1), dict(dtype=5),
                dict(batch=1 << 30)):
        assert attend(**bad) == 1, bad
    assert attend(width=257) == 3
    assert lib.tg_page_copy(6, 1, 4, None, None, None, None, 1, None, None) == 1
    assert lib.tg_page_copy(8, 1, 4, None, None, None, None, 0, None, None) == 0
    import ctypes

    from tensorgrad_b200.ops.paged import _FEW_PAIRS

    assert 0 < _FEW_PAIRS <= lib.tg_page_copy_few_max()
    ids = (ctypes.c_int64 * 2)(0, 4)
    at = ctypes.addressof(ids)
    assert lib.tg_page_copy_few(8, 1, 4, None, None, at, at + 8, 1, None) == 4
    assert lib.tg_page_copy_few(8, 1, 4, None, None, at + 8, at, 1, None) == 4
    assert lib.tg_page_copy_few(8, 1, 4, None, None, None, None, 65, None) == 1
    assert lib.tg_page_copy_few(8, 1, 4, None, None, None, None, 0, None) == 0
    assert lib.tg_paged_gather(0, 1 << 10, 1 << 20, 1, 1, None, None, 1, 1 << 20, None, 1, None,
                               None, None, None, None) == 1
    assert lib.tg_paged_gather(0, 1, 1, 1, 1, None, None, 1, 1 << 20, None, 1 << 11, None, None,
                               None, None, None) == 1
    assert lib.tg_paged_gather(0, 1, -1, 1, 1, None, None, 1, 1, None, 1, None, None, None, None,
                               None) == 1


class _Books:
    """A PagedKVCache whose pools are host arrays, to test the bookkeeping."""

    @staticmethod
    def make(monkeypatch, **sizes):
        import tensorgrad_b200.nn.paged as paged

        def copy(keys, values, src, dst):
            src, dst = np.asarray(src), np.asarray(dst)
            assert len(set(dst.tolist())) == len(dst) and not set(src) & set(dst)
            for pool in (keys, values):
                pool.data[:, dst] = pool.data[:, src]

        class Host:
            def __init__(self, shape):
                self.data = np.full(shape, np.nan)

        class Cache(paged.PagedKVCache):
            def _allocate(self, shape):
                return Host(shape), Host(shape)

            def _carry(self, old, new, pages):
                new.data[:, :pages] = old.data[:, :pages]

        monkeypatch.setattr(paged, "copy_pages", copy)
        return Cache(**sizes)


def _write(cache, seq, values):
    """Append a number per position to a sequence's pages, as a step does."""
    cache.reserve([seq], len(values))
    n = cache.length(seq)
    for i, v in enumerate(values):
        page = cache.pages(seq)[(n + i) // cache.page_size]
        cache.keys.data[:, page, :, (n + i) % cache.page_size] = v
    cache._get(seq).length += len(values)


def _read(cache, seq):
    out = [cache.keys.data[0, cache.pages(seq)[i // cache.page_size], 0, i % cache.page_size, 0]
           for i in range(cache.length(seq))]
    return out


@pytest.mark.parametrize("seed", range(6))
def test_paged_cache_books_hold_under_random_use(monkeypatch, seed):
    rng = np.random.default_rng(seed)
    cache = _Books.make(monkeypatch, layers=2, kv_heads=1, head_dim=2, num_pages=24,
                        page_size=int(rng.integers(1, 6)))
    model: dict[int, list[float]] = {}
    for step in range(400):
        what = rng.choice(["add", "fork", "free", "write", "write", "write", "compact", "resize"])
        seq = int(rng.choice(list(model))) if model else None
        if what == "add" and len(model) < 8:
            model[cache.add()] = []
        elif seq is None:
            continue
        elif what == "fork" and len(model) < 8:
            new = cache.fork(seq)
            model[new] = list(model[seq])
        elif what == "free":
            cache.free(seq)
            del model[seq]
        elif what == "write":
            new = [float(1000 * step + i) for i in range(rng.integers(0, 9))]
            before = (cache.pages_in_use, {s: cache.pages(s) for s in model})
            try:
                _write(cache, seq, new)
                model[seq] += new
            except MemoryError:
                assert before == (cache.pages_in_use, {s: cache.pages(s) for s in model})
        elif what == "compact":
            used = cache.compact()
            assert used == cache.pages_in_use
            assert all(p < used for s in model for p in cache.pages(s))
        elif what == "resize":
            n = int(rng.integers(1, 30))
            try:
                cache.resize(n)
                assert cache.num_pages == n
            except ValueError:
                assert cache.compact() > n
        held = [set(cache.pages(s)) for s in model]
        assert len(set().union(*held)) == cache.pages_in_use
        for s, values in model.items():
            assert cache.length(s) == len(values) and _read(cache, s) == values


def test_paged_cache_refusals_and_sharing(monkeypatch):
    cache = _Books.make(monkeypatch, layers=1, kv_heads=1, head_dim=1, num_pages=4, page_size=2)
    a = cache.add()
    _write(cache, a, [1.0, 2.0, 3.0])
    b, c = cache.fork(a), cache.fork(a)
    assert cache.pages_in_use == 2 and cache.pages(a) == cache.pages(b)
    cache.reserve([a, b], 1)  # a full page stays shared; a and b each copy, c keeps the old one
    assert cache.pages_in_use == 4
    assert len({cache.pages(s)[1] for s in (a, b, c)}) == 3
    assert len({cache.pages(s)[0] for s in (a, b, c)}) == 1
    with pytest.raises(MemoryError, match="free"):
        cache.reserve([a], 3)
    with pytest.raises(ValueError, match="twice"):
        cache.reserve([a, a], 1)
    with pytest.raises(KeyError, match="no sequence 77"):
        cache.free(77)
    with pytest.raises(ValueError, match="twice"):
        cache.batch([a, a])
    with pytest.raises(KeyError):
        cache.batch([78])
    with pytest.raises(ValueError, match="at least one"):
        cache.batch([])
    with pytest.raises(ValueError, match="in use"):
        cache.resize(1)
    for bad in (dict(layers=0), dict(page_size=0), dict(num_pages=-1)):
        with pytest.raises(ValueError, match="must be positive"):
            _Books.make(monkeypatch, **{**dict(layers=1, kv_heads=1, head_dim=1, num_pages=1,
                                               page_size=1), **bad})


# ---------------------------------------------------------------------- 8-bit integers
def _weight(outer, inner, dtype=np.float32):
    from tensorgrad_b200.ops import Int8Weight

    w = Int8Weight.__new__(Int8Weight)
    w.q, w.scale, w.in_features = _Meta((outer, -(-inner // 16) * 16), np.int8), _Meta((outer,), dtype), inner
    return w


def test_int8_ops_refuse_bad_arguments():
    from tensorgrad_b200.ops import Int8Weight, int8_linear, quantize_int8

    with pytest.raises(TypeError, match="takes an Int8Weight"):
        int8_linear(_t((2, 8)), _t((4, 8)))
    for shape in ((2, 7), ()):
        with pytest.raises(ValueError, match="does not match weight"):
            int8_linear(_t(shape), _weight(4, 8))
    with pytest.raises(TypeError, match="int64"):
        int8_linear(_t((2, 8), np.int64), _weight(4, 8))
    with pytest.raises(ValueError, match=r"bias \(3,\) for 4"):
        int8_linear(_t((2, 8)), _weight(4, 8), _t((3,)))
    learnt = _t((2, 8))
    learnt._requires_grad = True
    with pytest.raises(ValueError, match="inference"):
        int8_linear(learnt, _weight(4, 8))
    for shape in ((), (3, 0)):
        with pytest.raises(ValueError, match="last axis"):
            quantize_int8(_t(shape))
    with pytest.raises(TypeError, match="expected int8"):
        Int8Weight(_t((4, 16), np.float32), _t((4,)))
    with pytest.raises(TypeError, match="expected int8"):
        Int8Weight(_t((16,), np.int8), _t((4,)))
    for inner in (0, 17):
        with pytest.raises(ValueError, match=r"in_features must be in \[1, 16\]"):
            Int8Weight(_t((4, 16), np.int8), _t((4,)), inner)
    with pytest.raises(ValueError, match="4 floating scales"):
        Int8Weight(_t((4, 16), np.int8), _t((3,)))
    with pytest.raises(ValueError, match="4 floating scales"):
        Int8Weight(_t((4, 16), np.int8), _t((4,), np.int64))
    with pytest.raises(ValueError, match="expected a weight"):
        Int8Weight.quantize(_t((4,)))


def test_int8_entry_points_refuse_bad_sizes():
    from tensorgrad_b200._lib import lib

    def linear(rows=2, inner=20, ld=32, outer=3, dtype=0, scratch=None):
        return lib.tg_int8_linear(dtype, None, rows, inner, None, ld, None, None, None, outer,
                                  scratch, None)

    assert linear(rows=0) == 0 and linear(outer=0) == 0
    for bad in (dict(rows=-1), dict(inner=0), dict(ld=16), dict(ld=40), dict(outer=-1), dict()):
        assert linear(**bad) == 1, bad
    assert linear(inner=131073, ld=131088) == 3
    assert lib.tg_int8_quantize_rows(0, None, 1, 20, None, 19, None, None) == 1
