"""The key-value cache in pages: writing, gathering and copying pages, and the attention of one
new token over them (no counterpart in the reference, whose cache is contiguous:
nn/attention.py:27-111).

A pool of keys and one of values each hold ``(num_pages, kv_heads, page_size, head_dim)``; a
page table ``(batch, max_pages)`` names each sequence's pages in order, ``lengths`` ``(batch,)``
how many positions it holds. Tables and lengths are int64, on the host (checked there) or on
the device, where the kernels check them: an id or a length outside the cache raises
``IndexError`` at the next host synchronisation, as for device-resident ids elsewhere. All of it
is inference only and writes or reads in place; nothing is recorded for a backward pass.
``nn.PagedKVCache`` keeps the books (which pages belong to whom) on top.
"""

from __future__ import annotations

from typing import Any

import numpy as np

from tensorgrad_b200 import device
from tensorgrad_b200._lib import check, lib
from tensorgrad_b200.autograd import is_grad_enabled
from tensorgrad_b200.device import DeviceArray, dtype_code
from tensorgrad_b200.ops._util import as_tensor
from tensorgrad_b200.profiler import profiled
from tensorgrad_b200.tensor import Tensor

__all__ = ["append_pages", "copy_pages", "gather_pages", "paged_attention"]

_FEW_PAIRS = 64  # at most tg_page_copy_few_max(): their ids travel with the launch


def _inference_only(what: str, *tensors: Tensor) -> None:
    if is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} is for inference: use no_grad() or detach its inputs")


def _pools(what: str, keys: Any, values: Any, ndim: tuple[int, ...] = (4,)) -> tuple[Tensor, Tensor]:
    """The two pools: tensors of one shape and floating type with pages on axis -4."""
    for name, pool in (("key", keys), ("value", values)):
        if not isinstance(pool, Tensor):
            raise TypeError(f"{what}: the {name} pool must be a tensor (it is used in place), got "
                            f"{type(pool).__name__}")
    if keys.ndim not in ndim or 0 in keys.shape:
        raise ValueError(f"{what}: expected pools ({'layers, ' if 5 in ndim else ''}num_pages, "
                         f"kv_heads, page_size, head_dim), got {keys.shape}")
    if keys.shape != values.shape or keys.dtype != values.dtype:
        raise ValueError(f"{what}: key pool {keys.dtype} {keys.shape} and value pool "
                         f"{values.dtype} {values.shape} differ")
    dtype_code(keys.dtype)
    return keys, values


def _table(what: str, pages: Any, lengths: Any, batch: int, num_pages: int, page_size: int,
           extra: int = 0) -> tuple[DeviceArray, DeviceArray, int | None]:
    """Page table and lengths on the device as int64, and the flag word of their check there
    (None where the host has checked both). ``extra``: positions about to be written."""
    given = [x.data if isinstance(x, Tensor) else x for x in (pages, lengths)]
    table, held = (x if isinstance(x, DeviceArray) else np.asarray(x) for x in given)
    for name, x in (("pages", table), ("lengths", held)):
        if x.dtype.kind not in "iu":
            raise TypeError(f"{what}: {name} must be integers, got {x.dtype}")
        if isinstance(x, DeviceArray) and x.dtype != np.int64:
            raise TypeError(f"{what}: {name} on the device must be int64, got {x.dtype}")
    # As int64 before any arithmetic: lengths of a narrow type could wrap when `extra` is added.
    table, held = (x.astype(np.int64, copy=False) if isinstance(x, np.ndarray) else x
                   for x in (table, held))
    if len(table.shape) != 2 or table.shape[0] != batch or table.shape[1] == 0:
        raise ValueError(f"{what}: expected pages ({batch}, max_pages), got {table.shape}")
    if tuple(held.shape) != (batch,):
        raise ValueError(f"{what}: expected lengths ({batch},), got {held.shape}")
    if isinstance(held, np.ndarray):
        most = table.shape[1] * page_size
        if batch and (held.min() < 0 or held.max() + extra > most):
            raise IndexError(f"{what}: lengths must be in [0, {most - extra}] for a table of "
                             f"{table.shape[1]} pages of {page_size} positions")
        if isinstance(table, np.ndarray):
            used = np.arange(table.shape[1])[None] * page_size < held[:, None] + extra
            ids = table[used]
            if ids.size and (ids.min() < 0 or ids.max() >= num_pages):
                raise IndexError(f"{what}: page ids must be in [0, {num_pages})")
    checked = isinstance(table, np.ndarray) and isinstance(held, np.ndarray)
    out = [device.from_numpy(np.ascontiguousarray(x)) if isinstance(x, np.ndarray) else x
           for x in (table, held)]
    bad = None if checked else device.async_error_word(device.ASYNC_CACHE_PAGE)
    return out[0], out[1], bad


def append_strided(batch: int, tokens: int, k: tuple[int, tuple[int, int, int]],
                   v: tuple[int, tuple[int, int, int]], keys: DeviceArray, values: DeviceArray,
                   table: DeviceArray, lengths: DeviceArray, bad: int | None) -> None:
    """:func:`append_pages` on checked arguments, ``k`` and ``v`` as an address with element
    strides of (batch, head, position)."""
    num_pages, heads, size, width = keys.shape
    check(lib.tg_paged_append(dtype_code(keys.dtype), batch, tokens, heads, width, k[0], *k[1],
                              v[0], *v[1], keys.ptr, values.ptr, num_pages, size, table.ptr,
                              table.shape[1], lengths.ptr, bad, device.stream()), "append_pages")


@profiled("append_pages")
def append_pages(k: Any, v: Any, keys: Tensor, values: Tensor, pages: Any, lengths: Any) -> None:
    """Write new positions' keys and values ``(batch, kv_heads, tokens, head_dim)`` to the pools
    at positions ``lengths[b] .. lengths[b] + tokens - 1`` of each sequence, in place.

    ``lengths`` are those before the call and stay as they are. Sequences may share pages only
    below their lengths: a page that two sequences write to would hold either's values."""
    tk, tv = as_tensor(k), as_tensor(v)
    pk, pv = _pools("append_pages", keys, values)
    num_pages, heads, size, width = pk.shape
    if tk.ndim != 4 or tk.shape != tv.shape or (tk.shape[1], tk.shape[3]) != (heads, width):
        raise ValueError(f"append_pages: keys {tk.shape} and values {tv.shape} do not match "
                         f"pools {pk.shape}")
    if tk.dtype != pk.dtype or tv.dtype != pk.dtype:
        raise TypeError(f"append_pages: keys {tk.dtype} and values {tv.dtype} for pools of "
                        f"{pk.dtype}")
    _inference_only("append_pages", tk, tv, pk, pv)
    batch, _, tokens, _ = tk.shape
    table, held, bad = _table("append_pages", pages, lengths, batch, num_pages, size, tokens)
    strides = (heads * tokens * width, tokens * width, width)
    append_strided(batch, tokens, (tk.data.ptr, strides), (tv.data.ptr, strides), pk.data,
                   pv.data, table, held, bad)


@profiled("gather_pages")
def gather_pages(keys: Tensor, values: Tensor, pages: Any, lengths: Any,
                 longest: int) -> tuple[Tensor, Tensor]:
    """Each sequence's keys and values as contiguous ``(batch, kv_heads, longest, head_dim)``:
    positions below ``lengths[b]`` in order, zeros behind them."""
    pk, pv = _pools("gather_pages", keys, values)
    num_pages, heads, size, width = pk.shape
    batch = _rows_of(lengths)
    if longest < 0:
        raise ValueError(f"gather_pages: longest must not be negative, got {longest}")
    _inference_only("gather_pages", pk, pv)
    table, held, bad = _table("gather_pages", pages, lengths, batch, num_pages, size)
    out = [device.empty((batch, heads, longest, width), pk.dtype) for _ in range(2)]
    check(lib.tg_paged_gather(dtype_code(pk.dtype), batch, longest, heads, width, pk.data.ptr,
                              pv.data.ptr, num_pages, size, table.ptr, table.shape[1], held.ptr,
                              out[0].ptr, out[1].ptr, bad, device.stream()), "gather_pages")
    return Tensor._wrap(out[0]), Tensor._wrap(out[1])


def _rows_of(lengths: Any) -> int:
    shape = lengths.shape if isinstance(lengths, Tensor | DeviceArray) else np.shape(lengths)
    if len(shape) != 1:
        raise ValueError(f"expected lengths (batch,), got shape {tuple(shape)}")
    return shape[0]


@profiled("copy_pages")
def copy_pages(keys: Tensor, values: Tensor, src: Any, dst: Any) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in both pools, in place: pools
    ``(num_pages, ...)`` as above or ``(layers, num_pages, ...)``, where every layer's page
    moves. ``src`` and ``dst`` are host integers; a page may be copied to several, but each
    destination is written once and is not a source of the same call."""
    pk, pv = _pools("copy_pages", keys, values, (4, 5))
    _inference_only("copy_pages", pk, pv)
    a, b = np.asarray(src), np.asarray(dst)
    if a.ndim != 1 or a.shape != b.shape:
        raise ValueError(f"copy_pages: expected lists of as many sources as destinations, got "
                         f"{a.shape} and {b.shape}")
    n = a.size
    if n == 0:
        return
    if a.dtype.kind not in "iu" or b.dtype.kind not in "iu":
        raise TypeError(f"copy_pages: page ids must be integers, got {a.dtype} and {b.dtype}")
    layers = pk.shape[0] if pk.ndim == 5 else 1
    num_pages, heads, size, width = pk.shape[-4:]
    pairs = np.empty((2, n), dtype=np.int64)
    pairs[0], pairs[1] = a, b
    if pairs.min() < 0 or pairs.max() >= num_pages:
        raise IndexError(f"copy_pages: page ids must be in [0, {num_pages})")
    few = n <= _FEW_PAIRS
    if few:
        to = set(pairs[1].tolist())
        distinct, apart = len(to) == n, to.isdisjoint(pairs[0].tolist())
    else:
        written = np.zeros(num_pages, dtype=np.bool_)
        written[pairs[1]] = True
        distinct, apart = np.count_nonzero(written) == n, not written[pairs[0]].any()
    if not distinct:
        raise ValueError("copy_pages: a destination page is given twice")
    if not apart:
        raise ValueError("copy_pages: a page is both a source and a destination")
    where = (heads * size * width * pk.dtype.itemsize, layers, num_pages, pk.data.ptr, pv.data.ptr)
    if few:
        at = pairs.ctypes.data
        check(lib.tg_page_copy_few(*where, at, at + 8 * n, n, device.stream()), "copy_pages")
        return
    ids = device.from_numpy(pairs)
    check(lib.tg_page_copy(*where, ids.ptr, ids.ptr + 8 * n, n, None, device.stream()),
          "copy_pages")


def attend_strided(batch: int, heads: int, q: tuple[int, tuple[int, int]], keys: DeviceArray,
                   values: DeviceArray, table: DeviceArray, lengths: DeviceArray, longest: int,
                   out: DeviceArray, lse: DeviceArray | None, bad: int | None) -> None:
    """:func:`paged_attention` on checked arguments, ``q`` as an address with element strides
    of (batch, head)."""
    num_pages, kv_heads, size, width = keys.shape
    code = dtype_code(keys.dtype)
    nbytes = lib.tg_paged_attention_scratch_bytes(code, batch, heads, kv_heads, width, longest)
    scratch = device.scratch(nbytes) if nbytes > 16 else None
    check(lib.tg_paged_attention(
        code, batch, heads, kv_heads, width, q[0], *q[1], keys.ptr, values.ptr, num_pages, size,
        table.ptr, table.shape[1], lengths.ptr, longest, out.ptr,
        None if lse is None else lse.ptr, bad, None if scratch is None else scratch.ptr,
        device.stream()), "paged_attention")


@profiled("paged_attention")
def paged_attention(q: Any, keys: Tensor, values: Tensor, pages: Any, lengths: Any, *,
                    longest: int | None = None,
                    return_lse: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``softmax(q k^T / sqrt(d)) v`` of one new token per sequence: queries ``(batch, heads,
    head_dim)`` over the first ``lengths[b]`` positions of the sequence's pages (its own key
    among them, once appended). ``heads`` is a multiple of the pools' key heads; query head
    ``h`` reads key head ``h // (heads // kv_heads)``. ``head_dim`` is at most 256.

    A sequence of length 0 gives zeros (and a log-sum-exp of ``-inf``). ``longest`` may say
    about how long the longest sequence is, where the table is much wider: the work is split
    accordingly. With ``return_lse`` also the log-sum-exp of the scaled scores
    ``(batch, heads)``, with which results over parts of a sequence can be joined."""
    tq = as_tensor(q)
    pk, pv = _pools("paged_attention", keys, values)
    num_pages, kv_heads, size, width = pk.shape
    if tq.ndim != 3 or tq.shape[2] != width or tq.shape[1] == 0 or tq.shape[1] % kv_heads:
        raise ValueError(f"paged_attention: queries {tq.shape} do not match pools {pk.shape}")
    if width > 256:
        raise NotImplementedError(f"paged_attention: head_dim {width} (at most 256)")
    if tq.dtype != pk.dtype:
        raise TypeError(f"paged_attention: queries {tq.dtype} for pools of {pk.dtype}")
    _inference_only("paged_attention", tq, pk, pv)
    batch, heads, _ = tq.shape
    table, held, bad = _table("paged_attention", pages, lengths, batch, num_pages, size)
    if longest is None:
        longest = table.shape[1] * size
        host = lengths.data if isinstance(lengths, Tensor) else lengths
        if batch and not isinstance(host, DeviceArray):
            longest = int(np.max(host))
    elif longest < 0:
        raise ValueError(f"paged_attention: longest must not be negative, got {longest}")
    out = device.empty(tq.shape, pk.dtype)
    lse = device.empty((batch, heads), pk.dtype) if return_lse else None
    attend_strided(batch, heads, (tq.data.ptr, (heads * width, width)), pk.data, pv.data, table,
                   held, max(longest, 1), out, lse, bad)
    return Tensor._wrap(out) if lse is None else (Tensor._wrap(out), Tensor._wrap(lse))
