"""The paged key-value cache on the device: page operations bit for bit against NumPy, the
attention of one new token against its definition in extended precision, and the model path
(ragged batches, forks, continued prompts) against the contiguous one.

Tolerance of the attention: a score is a dot product of d terms and a scaling, off by at most
(d + 2) h sum|q_i k_i| / sqrt(d) absolutely (h half a step of the type, ties to the worst
summation order), which moves its weight by the same relative amount; the exponential adds 4 h
(8 h with its argument's rounding at 2 h per unit of its size), and n weighted values are then
summed with at most n + 2 roundings, again over the absolute values. The output's error is
bounded by the sum over positions of p_i |v_i| times all of that, twice (numerator and sum).
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[np.float32, np.float64], ids=["fp32", "fp64"])
def dtype(request):
    return request.param


def _cache(rng, dtype, lengths, kv_heads, width, size, spare=2):
    """Pools of noise, a table of shuffled pages (junk behind each sequence's last page)."""
    lengths = np.asarray(lengths, dtype=np.int64)
    per = max(1, int(-(-lengths.max() // size))) + 1
    num = len(lengths) * per + spare
    pools = [rng.standard_normal((num, kv_heads, size, width)).astype(dtype) for _ in range(2)]
    table = rng.permutation(num)[:len(lengths) * per].reshape(len(lengths), per)
    for b, n in enumerate(lengths):
        table[b, -(-n // size):] = -7  # never read
    return pools[0], pools[1], table.astype(np.int64), lengths


def _rows(pool, table, n):
    size = pool.shape[2]
    pages = table[:-(-n // size)]
    return np.concatenate([pool[p] for p in pages], axis=1)[:, :n] if n else pool[0][:, :0]


def _attention(q, keys, values, table, lengths):
    """(out, lse, bound on out's error / h) in extended precision."""
    b, heads, d = q.shape
    kv_heads = keys.shape[1]
    g = heads // kv_heads
    out = np.zeros(q.shape, np.longdouble)
    bound = np.zeros(q.shape, np.longdouble)
    lse = np.full((b, heads), -np.inf, np.longdouble)
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        k = _rows(keys, table[i], n).astype(np.longdouble)
        v = _rows(values, table[i], n).astype(np.longdouble)
        for h in range(heads):
            x = q[i, h].astype(np.longdouble)
            s = k[h // g] @ x / np.sqrt(np.longdouble(d))
            size = np.abs(k[h // g]) @ np.abs(x) / np.sqrt(np.longdouble(d))
            m = s.max()
            e = np.exp(s - m)
            p = e / e.sum()
            out[i, h] = p @ v[h // g]
            lse[i, h] = m + np.log(e.sum())
            off = (d + 4) * size + 2 * (m - s) + 8 + 2 * np.abs(m) + (n + 4)
            mean_off = p @ off
            bound[i, h] = (p * (off + mean_off)) @ np.abs(v[h // g]) + np.abs(out[i, h])
    return out, lse, bound


CASES = [
    # lengths, heads, kv_heads, width, page size
    ([1], 1, 1, 64, 16),
    ([17, 0, 1, 16], 12, 12, 64, 16),
    ([100, 33, 0, 257, 64], 8, 2, 128, 16),
    ([5, 700], 6, 3, 40, 5),
    ([31, 32, 33], 4, 4, 33, 7),
    ([1000, 3], 8, 1, 256, 32),
    ([2500, 1, 900], 3, 1, 16, 64),
    ([300], 10, 2, 80, 1),
    ([129, 40], 16, 1, 96, 100),
    ([50, 2], 7, 1, 1, 3),
    ([777], 24, 2, 255, 9),
    ([4000, 4096, 12], 4, 2, 8, 16),
    ([900, 33, 0, 5000], 10, 2, 128, 16),
    ([200] * 9, 64, 8, 64, 8),
    ([3000, 2], 24, 3, 33, 16),
]


@pytest.mark.parametrize("lengths,heads,kv_heads,width,size", CASES)
def test_attention_matches_definition(lengths, heads, kv_heads, width, size, dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(sum(lengths) + heads + width)
    keys, values, table, held = _cache(rng, dtype, lengths, kv_heads, width, size)
    q = (2 * rng.standard_normal((len(lengths), heads, width))).astype(dtype)
    out, lse = tg.paged_attention(tg.Tensor(q), tg.Tensor(keys), tg.Tensor(values), table, held,
                                  return_lse=True)
    ref, ref_lse, bound = _attention(q, keys, values, table, held)
    h = np.finfo(dtype).eps / 2
    assert out.dtype == dtype and out.shape == q.shape
    assert np.all(np.abs(out.numpy() - ref) <= bound * h)
    empty = held == 0
    assert np.all(out.numpy()[empty] == 0) and np.all(np.isneginf(lse.numpy()[empty]))
    full = ~empty
    scale = (width + 6 + max(lengths)) * h * (8 + np.abs(ref_lse[full]).astype(np.float64).max())
    assert np.all(np.abs(lse.numpy()[full] - ref_lse[full]) <= 2 * scale)


@pytest.mark.parametrize("heads,kv_heads,width", [(1, 1, 64), (8, 2, 128), (8, 1, 40)])
@pytest.mark.parametrize("course", ["rises", "falls", "creeps", "leaps"])
def test_attention_where_the_maximum_moves(course, heads, kv_heads, width, dtype):
    """Scores that climb or fall by tens, by less than one in all, or in steps of some hundred."""
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(width)
    keys, values, table, held = _cache(rng, dtype, [900, 70], kv_heads, width, 16)
    u = rng.choice([-1.0, 1.0], width)
    t = np.linspace(0, 1, 900)
    reach = {"rises": 60 * t, "falls": 60 * (1 - t), "creeps": t,
             "leaps": 150 * np.floor(5 * t)}[course]
    for b, n in enumerate(held):
        for at in range(n):
            row = keys[table[b, at // 16], :, at % 16]
            row *= 0.25
            row += (reach[at] / np.sqrt(width) * u).astype(dtype)
    q = (u + 0.25 * rng.standard_normal((2, heads, width))).astype(dtype)
    out = tg.paged_attention(tg.Tensor(q), tg.Tensor(keys), tg.Tensor(values), table, held)
    ref, _, bound = _attention(q, keys, values, table, held)
    assert np.all(np.abs(out.numpy() - ref) <= bound * np.finfo(dtype).eps / 2)


def test_device_tables_hints_and_views_give_the_same(dtype):
    import tensorgrad_b200 as tg
    from tensorgrad_b200 import device

    rng = np.random.default_rng(2)
    keys, values, table, held = _cache(rng, dtype, [3000, 1, 0, 640], 2, 64, 16)
    q = rng.standard_normal((4, 4, 64)).astype(dtype)
    host = tg.paged_attention(tg.Tensor(q), tg.Tensor(keys), tg.Tensor(values), table, held)
    ref, _, bound = _attention(q, keys, values, table, held)
    h = np.finfo(dtype).eps / 2
    on_device = tg.Tensor(table), tg.Tensor(held)
    for longest in (None, 1, 640, 3000, 10**6):
        got = tg.paged_attention(tg.Tensor(q), tg.Tensor(keys), tg.Tensor(values), *on_device,
                                 longest=longest)
        assert np.all(np.abs(got.numpy() - ref) <= bound * h), longest
    # Pools and queries that start one element off a 16-byte boundary.
    views = []
    for a in (q, keys, values):
        flat = device.from_numpy(np.concatenate([np.zeros(1, dtype), a.reshape(-1)]))
        views.append(tg.Tensor._wrap(flat.flat_view(1, a.size, a.shape)))
    got = tg.paged_attention(*views, table, held)
    assert np.all(np.abs(got.numpy() - ref) <= bound * h)
    assert np.all(np.abs(host.numpy() - ref) <= bound * h)


def test_parts_join_by_their_log_sum_exp():
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(5)
    keys, values, table, held = _cache(rng, np.float64, [96], 2, 32, 16)
    q = tg.Tensor(rng.standard_normal((1, 4, 32)))
    pools = tg.Tensor(keys), tg.Tensor(values)
    whole = tg.paged_attention(q, *pools, table, held).numpy()
    a, la = (x.numpy() for x in tg.paged_attention(q, *pools, table[:, :2], [32], return_lse=True))
    b, lb = (x.numpy() for x in tg.paged_attention(q, *pools, table[:, 2:], [64], return_lse=True))
    w = 1 / (1 + np.exp(lb - la))[..., None]
    np.testing.assert_allclose(a * w + b * (1 - w), whole, rtol=0, atol=1e-13)


def test_values_behind_the_end_do_not_matter(dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(8)
    keys, values, table, held = _cache(rng, dtype, [19, 5], 1, 64, 16)
    q = rng.standard_normal((2, 2, 64)).astype(dtype)
    first = tg.paged_attention(tg.Tensor(q), tg.Tensor(keys), tg.Tensor(values), table, held).numpy()
    for b, n in enumerate(held):
        keys[table[b, n // 16], :, n % 16:] = np.nan
        values[table[b, n // 16], :, n % 16:] = np.inf
    again = tg.paged_attention(tg.Tensor(q), tg.Tensor(keys), tg.Tensor(values), table, held).numpy()
    np.testing.assert_array_equal(first, again)


def test_bad_device_pages_raise_at_the_next_synchronisation():
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(1)
    keys, values, table, held = _cache(rng, np.float32, [40, 20], 2, 64, 16)
    q = tg.Tensor(rng.standard_normal((2, 2, 64)).astype(np.float32))
    pools = tg.Tensor(keys), tg.Tensor(values)
    wrong = table.copy()
    wrong[0, 1] = len(keys)
    for pages, lengths in ((wrong, held), (table, np.array([40, -3])), (table, np.array([10**6, 1]))):
        out = tg.paged_attention(q, *pools, tg.Tensor(pages), tg.Tensor(lengths))
        with pytest.raises(IndexError, match="paged cache"):
            out.numpy()
        got = tg.gather_pages(*pools, tg.Tensor(pages), tg.Tensor(lengths), 8)
        if pages is table:
            with pytest.raises(IndexError, match="paged cache"):
                got[0].numpy()
        else:
            got[0].numpy()  # only the first page is read
    k = tg.Tensor(np.ones((2, 2, 3, 64), np.float32))
    tg.append_pages(k, k, *pools, tg.Tensor(wrong), tg.Tensor(np.array([30, 0])))
    with pytest.raises(IndexError, match="paged cache"):
        tg.synchronize()
    # What could be written was; the rest of the pool is as it was.
    after = pools[0].numpy()
    expect = keys.copy()
    expect[table[0, 2], :, 0] = 1  # positions 30 and 31 lie on the bad page, 32 on the next
    expect[table[1, 0], :, :3] = 1
    np.testing.assert_array_equal(after, expect)


@pytest.mark.parametrize("tokens,kv_heads,width,size", [(1, 12, 64, 16), (5, 3, 40, 4),
                                                        (33, 2, 33, 7), (1, 1, 1, 1),
                                                        (300, 2, 128, 16)])
def test_append_then_gather(tokens, kv_heads, width, size, dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(tokens + width)
    start = np.array([0, 3, size, 2 * size - 1, 20], dtype=np.int64)
    keys, values, table, held = _cache(rng, dtype, start + tokens, kv_heads, width, size)
    k, v = rng.standard_normal((2, 5, kv_heads, tokens, width)).astype(dtype)
    pools = tg.Tensor(keys), tg.Tensor(values)
    for lengths in (start, tg.Tensor(start)):
        pools = tg.Tensor(keys), tg.Tensor(values)
        pages = table if lengths is start else tg.Tensor(table)
        tg.append_pages(tg.Tensor(k), tg.Tensor(v), *pools, pages, lengths)
        expect = [keys.copy(), values.copy()]
        for b, n in enumerate(start):
            for t in range(tokens):
                for pool, new in zip(expect, (k, v), strict=True):
                    pool[table[b, (n + t) // size], :, (n + t) % size] = new[b, :, t]
        for pool, ref in zip(pools, expect, strict=True):
            np.testing.assert_array_equal(pool.numpy(), ref)
    longest = int(held.max()) + 2
    got = tg.gather_pages(*pools, table, held, longest)
    for g, pool in zip(got, expect, strict=True):
        ref = np.zeros((5, kv_heads, longest, width), dtype)
        for b, n in enumerate(held):
            ref[b, :, :n] = _rows(pool, table[b], n)
        np.testing.assert_array_equal(g.numpy(), ref)
    short = tg.gather_pages(*pools, table, held, 2)[0].numpy()
    np.testing.assert_array_equal(short, got[0].numpy()[:, :, :2])


@pytest.mark.parametrize("shape", [(6, 2, 4, 8), (3, 7, 1, 5, 3), (12, 40, 4, 16, 64),
                                   (128, 1, 16, 64), (2, 130, 1, 7, 33), (3, 400, 2, 16, 80),
                                   (5000, 1, 1, 1)])
def test_copy_pages(shape, dtype):
    import tensorgrad_b200 as tg

    rng = np.random.default_rng(shape[0])
    keys, values = rng.standard_normal((2, *shape)).astype(dtype)
    n = shape[-4]
    order = rng.permutation(n)
    dst, src = order[:n // 2], rng.choice(order[n // 2:], n // 2)  # a source may repeat
    pools = tg.Tensor(keys), tg.Tensor(values)
    tg.copy_pages(*pools, src, dst)
    for pool, ref in zip(pools, (keys, values), strict=True):
        at = ref if ref.ndim == 4 else np.moveaxis(ref, 1, 0)
        at[dst] = at[src]
        np.testing.assert_array_equal(pool.numpy(), ref)


def test_pools_beyond_32_bit_offsets():
    import tensorgrad_b200 as tg
    from tensorgrad_b200 import device

    num = 2**32 // (16 * 64) + 8  # more than 2^32 elements in a pool
    rng = np.random.default_rng(3)
    pools = [tg.Tensor._wrap(device.empty((num, 1, 16, 64), np.float32)) for _ in range(2)]
    table = np.array([[num - 1, num - 4], [5, num - 2]])
    k, v = rng.standard_normal((2, 2, 1, 20, 64)).astype(np.float32)
    tg.append_pages(tg.Tensor(k), tg.Tensor(v), *pools, table, [0, 0])
    held = np.array([20, 20])
    for got, ref in zip(tg.gather_pages(*pools, table, held, 20), (k, v), strict=True):
        np.testing.assert_array_equal(got.numpy(), ref)
    q = rng.standard_normal((2, 3, 64)).astype(np.float32)
    first = tg.paged_attention(tg.Tensor(q), *pools, table, held).numpy()
    small = [np.stack([x[b, 0].reshape(-1) for b in range(2)]).reshape(2, 1, 20, 64)
             for x in (k, v)]
    ref = tg.paged_attention(tg.Tensor(q), tg.Tensor(small[0]), tg.Tensor(small[1]),
                             np.array([[0], [1]]), held).numpy()
    np.testing.assert_array_equal(first, ref)  # which lane has a position is the same
    tg.copy_pages(*pools, [num - 1, num - 4, 5], [7, num - 5, num - 6])
    moved = np.array([[7, num - 5], [num - 6, num - 2]])
    np.testing.assert_array_equal(tg.paged_attention(tg.Tensor(q), *pools, moved, held).numpy(),
                                  first)


# ---------------------------------------------------------------------- the model's path
def _model(dtype, block=48):
    import tensorgrad_b200 as tg

    tg.set_default_dtype(dtype)
    tg.manual_seed(3)
    model = tg.nn.GPT(tg.nn.GPTConfig(vocab_size=61, block_size=block, n_layer=2, n_head=4,
                                      n_embd=64))
    tg.set_default_dtype(np.float32)
    return model.eval()


def test_ragged_steps_forks_and_continued_prompts_match_the_full_forward(dtype):
    rng = np.random.default_rng(11)
    model = _model(dtype)
    tol = 1e-4 if dtype == np.float32 else 1e-10  # the framework's parity bar per type

    def full(ids):
        return model(np.array(ids)[None]).numpy()[0]

    def close(a, b):
        assert np.abs(a - b).max() <= tol * np.abs(b).max()

    cache = model.make_paged_cache(num_pages=40, page_size=5)
    texts = [rng.integers(0, 61, n).tolist() for n in (1, 7, 20)]
    seqs = [cache.add() for _ in texts]
    for s, t in zip(seqs, texts, strict=True):
        close(model(np.array(t)[None], cache=cache.batch([s])).numpy()[0], full(t))
    fork = cache.fork(seqs[1])
    texts.append(list(texts[1]))
    seqs.append(fork)
    for _ in range(4):  # one token each, at four different lengths
        new = rng.integers(0, 61, 4)
        for t, x in zip(texts, new, strict=True):
            t.append(int(x))
        got = model(new[:, None], cache=cache.batch(seqs)).numpy()[:, -1]
        for g, t in zip(got, texts, strict=True):
            close(g, full(t)[-1])
    before = cache.pages_in_use
    cache.free(seqs.pop(0))
    texts.pop(0)
    assert cache.compact() < before
    cache.resize(cache.pages_in_use + 12)
    more = rng.integers(0, 61, (3, 6))  # several tokens that continue ragged sequences
    for t, x in zip(texts, more, strict=True):
        t.extend(x.tolist())
    got = model(more, cache=cache.batch(seqs)).numpy()
    for g, t in zip(got, texts, strict=True):
        close(g, full(t)[-6:])
    assert [cache.length(s) for s in seqs] == [len(t) for t in texts]


def test_model_refuses_what_the_cache_cannot_hold():
    model = _model(np.float32)
    cache = model.make_paged_cache(num_pages=2, page_size=16)
    a = cache.add()
    with pytest.raises(MemoryError):
        model(np.zeros((1, 33), np.int64), cache=cache.batch([a]))
    with pytest.raises(ValueError, match="exceeds block_size 48"):
        model(np.zeros((1, 49), np.int64), cache=cache.batch([a]))
    with pytest.raises(ValueError, match="2 rows of ids for 1"):
        model(np.zeros((2, 3), np.int64), cache=cache.batch([a]))
    with pytest.raises(ValueError, match="at least one token"):
        model(np.zeros((1, 0), np.int64), cache=cache.batch([a]))
    with pytest.raises(ValueError, match="the model has"):
        _model(np.float64)(np.zeros((1, 3), np.int64), cache=cache.batch([a]))
    with pytest.raises(ValueError, match="call eval"):
        model.train()(np.zeros((1, 3), np.int64), cache=cache.batch([a]))
    assert cache.length(a) == 0 and cache.pages_in_use == 0


def test_generate_batch_matches_generate():
    rng = np.random.default_rng(0)
    model = _model(np.float64)
    prompts = [rng.integers(0, 61, n) for n in (3, 11, 1)]
    got = model.generate_batch(prompts, 9, samples=2, top_k=1, page_size=4)
    for p, pair in zip(prompts, got, strict=True):
        want = model.generate(p[None], 9, top_k=1)[0]
        for s in pair:
            np.testing.assert_array_equal(s.ids, want)
            logits = model(want[None]).numpy()[0]
            lp = logits - np.log(np.exp(logits).sum(-1, keepdims=True))
            at = np.arange(len(p) - 1, len(want) - 1)
            np.testing.assert_allclose(s.log_probs, lp[at, want[at + 1]], rtol=0, atol=1e-10)
    drawn = model.generate_batch(prompts, 5, samples=3, rng=np.random.default_rng(4))
    assert len({tuple(s.ids) for s in drawn[1]}) > 1
    assert model.generate_batch([], 5) == []
    assert model.generate_batch(prompts, 0)[2][0].ids.tolist() == prompts[2].tolist()
    with pytest.raises(ValueError, match="block_size"):
        model.generate_batch([np.zeros(40, int)], 9)
    with pytest.raises(ValueError, match="at least one id"):
        model.generate_batch([np.zeros(0, int)], 2)
