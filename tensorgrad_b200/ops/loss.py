"""Loss functions (the reference's ops/loss.py) and the scores of tokens under logits."""

from __future__ import annotations

import math
from typing import Any, Literal, NamedTuple

import numpy as np

from tensorgrad_b200 import device
from tensorgrad_b200._lib import check, lib
from tensorgrad_b200.autograd import is_grad_enabled
from tensorgrad_b200.device import DeviceArray, dtype_code
from tensorgrad_b200.ops import reduce
from tensorgrad_b200.ops._util import (
    Need, as_tensor, coerce_pair, graph_by_composite, make_result,
)
from tensorgrad_b200.ops.elementwise import cast_array
from tensorgrad_b200.profiler import profiled
from tensorgrad_b200.tensor import Tensor

__all__ = ["Reduction", "TokenLogProbs", "binary_cross_entropy_with_logits", "cross_entropy",
           "mse_loss", "token_log_probs"]

Reduction = Literal["mean", "sum", "none"]
_RED = {"mean": 0, "sum": 1, "none": 2}


@profiled("cross_entropy")
def cross_entropy(logits: Any, target: Any, *, ignore_index: int = -100,
                  reduction: Reduction = "mean") -> Tensor:
    """Softmax cross-entropy from unnormalised logits, class axis last (ops/loss.py:23-97).

    One kernel pass per row computes the log-sum-exp (online max and sum) and the row loss;
    the mean over non-ignored rows is a fixed-order float64 sum. The VJP is one pass writing
    ``(softmax - onehot) * g / n_valid``. Host targets are validated on the host, as the
    reference does, before any device work; device-resident targets are validated by the
    kernel and an out-of-range one raises at the next host synchronisation.
    """
    tl = as_tensor(logits)
    classes = tl.shape[-1]
    dev_t = target.data if isinstance(target, Tensor) else target
    bad = None
    if isinstance(dev_t, DeviceArray):
        # Device-resident targets stay on the device: the kernel checks them and an
        # out-of-range target raises IndexError at the next host synchronisation.
        if dev_t.dtype.kind not in "iu":
            raise TypeError(f"cross_entropy targets must be integers, got {dev_t.dtype}")
        if tl.shape[:-1] != dev_t.shape:
            raise ValueError(f"logits {tl.shape} and targets {dev_t.shape} are incompatible")
        if reduction not in _RED:
            raise ValueError(f"unknown reduction {reduction!r}")
        tgt = dev_t if dev_t.dtype == np.int64 else cast_array(dev_t, np.dtype(np.int64))
        t_shape = dev_t.shape
        bad = device.async_error_word(device.ASYNC_CLASS_TARGET)
    else:
        t = np.asarray(target)
        if not np.issubdtype(t.dtype, np.integer):
            raise TypeError(f"cross_entropy targets must be integers, got {t.dtype}")
        if tl.shape[:-1] != t.shape:
            raise ValueError(f"logits {tl.shape} and targets {t.shape} are incompatible")
        if reduction not in _RED:
            raise ValueError(f"unknown reduction {reduction!r}")
        flat_t = np.ascontiguousarray(t.reshape(-1), dtype=np.int64)
        valid = flat_t != ignore_index
        safe = np.where(valid, flat_t, 0)
        if np.any((safe < 0) | (safe >= classes)):
            raise IndexError(f"target out of range for {classes} classes")
        tgt = device.from_numpy(flat_t)
        t_shape = t.shape
    x = tl.data if tl.dtype.kind == "f" else cast_array(tl.data, np.dtype(np.float64))
    rows = tgt.size
    code = dtype_code(x.dtype)
    red = _RED[reduction]
    lse = device.empty((rows,), x.dtype)
    row_loss = device.empty((rows,), x.dtype)
    n_valid = device.empty((1,), np.int64)
    out = row_loss.reshape(t_shape) if red == 2 else device.empty((), x.dtype)
    check(lib.tg_cross_entropy_forward(code, x.ptr, tgt.ptr, lse.ptr, row_loss.ptr, out.ptr,
                                       rows, classes, ignore_index, red, n_valid.ptr, bad,
                                       device.stream()), "cross_entropy")

    def backward(g: DeviceArray, need: Need) -> tuple[DeviceArray]:
        if g.dtype != x.dtype:
            g = cast_array(g, x.dtype)
        grad = device.empty(tl.shape, x.dtype)
        check(lib.tg_cross_entropy_backward(code, x.ptr, tgt.ptr, lse.ptr, g.ptr, n_valid.ptr,
                                            grad.ptr, rows, classes, ignore_index, red,
                                            device.stream()), "cross_entropy backward")
        return (grad if grad.dtype == tl.dtype else cast_array(grad, tl.dtype),)

    host_targets = None if isinstance(dev_t, DeviceArray) else flat_t

    def graph(g: Tensor, y: Tensor, need: Need) -> tuple[Tensor]:
        # (softmax(x) - onehot) * valid * weight in differentiable ops: softmax as e / sum(e)
        # with e = exp(x - lse), the saved log-sum-exp a constant shift; the one-hot rows
        # (host targets) uploaded once.
        from tensorgrad_b200.ops.elementwise import exp, mul, sub
        from tensorgrad_b200.ops.shape import reshape

        if host_targets is None:
            raise NotImplementedError("create_graph=True: cross_entropy with device-resident "
                                      "targets has no differentiable VJP; pass host targets")
        keep = host_targets != ignore_index
        onehot = np.zeros((rows, classes), dtype=x.dtype)
        onehot[np.flatnonzero(keep), host_targets[keep]] = 1.0
        x2 = reshape(tl, (rows, classes))
        e = exp(sub(x2, Tensor._wrap(lse.reshape((rows, 1)))))
        probs = e / reduce.sum(e, axis=-1, keepdims=True)
        diff = mul(sub(probs, Tensor(onehot)), Tensor(keep.astype(x.dtype).reshape(rows, 1)))
        if red == 2:
            weight = reshape(g, (rows, 1))
        elif red == 0:
            weight = g / float(max(int(keep.sum()), 1))
        else:
            weight = g
        return (reshape(mul(diff, weight), tl.shape),)

    return make_result(out, (tl,), backward, "cross_entropy", graph)


@profiled("mse_loss")
def mse_loss(prediction: Any, target: Any, *, reduction: Reduction = "mean") -> Tensor:
    """``(prediction - target) ** 2`` reduced, composed as the reference composes it
    (ops/loss.py:148-161)."""
    tp, tt = coerce_pair(prediction, target)
    sq = (tp - tt) ** 2
    if reduction == "mean":
        return reduce.mean(sq)
    if reduction == "sum":
        return reduce.sum(sq)
    if reduction == "none":
        return sq
    raise ValueError(f"unknown reduction {reduction!r}")


@profiled("binary_cross_entropy")
def binary_cross_entropy_with_logits(logits: Any, target: Any, *,
                                     reduction: Reduction = "mean") -> Tensor:
    """Binary cross entropy of ``sigmoid(logits)`` against ``target`` in [0, 1]
    (ops/loss.py:100-145): ``max(z, 0) - z y + log1p(exp(-|z|))`` on the device, so nothing
    overflows; the gradient is ``sigmoid(z) - y`` for the logits and ``-z`` for the targets."""
    from tensorgrad_b200._lib import ABS, ADD, EXP, LOG1P, MUL, NEG, RELU, SIGMOID, SUB
    from tensorgrad_b200.ops.elementwise import _unary, binary_array, scale_array

    tz, ty = coerce_pair(logits, target)
    if tz.shape != ty.shape:
        raise ValueError(f"logits {tz.shape} and target {ty.shape} must have the same shape")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unknown reduction {reduction!r}")
    dt = np.result_type(tz.dtype, ty.dtype)
    if dt.kind != "f":
        dt = np.dtype(np.float64)
    z = tz.data if tz.dtype == dt else cast_array(tz.data, dt)
    y = ty.data if ty.dtype == dt else cast_array(ty.data, dt)
    softplus_tail = _unary(_unary(_unary(_unary(z, ABS), NEG), EXP), LOG1P)
    losses = binary_array(binary_array(_unary(z, RELU), binary_array(z, y, MUL), SUB),
                          softplus_tail, ADD)
    n = max(losses.size, 1)
    if reduction == "none":
        out = losses
    else:
        total = reduce.sum_array(losses, tuple(range(losses.ndim))).reshape(())
        out = scale_array(total, 1.0 / n) if reduction == "mean" else total
    scale = 1.0 / n if reduction == "mean" else 1.0

    def upstream_array(g: DeviceArray) -> DeviceArray:
        if reduction == "none":
            return g
        from tensorgrad_b200.ops.shape import broadcast_array

        return broadcast_array(scale_array(g, scale), z.shape)

    def backward(g: DeviceArray, need: Need) -> tuple[DeviceArray | None, DeviceArray | None]:
        up = upstream_array(g)
        return (binary_array(binary_array(_unary(z, SIGMOID), y, SUB), up, MUL)
                if need[0] else None,
                binary_array(_unary(z, NEG), up, MUL) if need[1] else None)

    def graph(g: Tensor, y_: Tensor, need: Need) -> tuple[Tensor | None, Tensor | None]:
        from tensorgrad_b200.ops.elementwise import sigmoid
        from tensorgrad_b200.ops.shape import broadcast_to

        up = g if reduction == "none" else broadcast_to(g * scale, tz.shape)
        return ((sigmoid(tz) - ty) * up if need[0] else None,
                -tz * up if need[1] else None)

    return make_result(out, (tz, ty), backward, "binary_cross_entropy", graph)


class TokenLogProbs(NamedTuple):
    """What :func:`token_log_probs` gives: per row the target's log probability and the
    entropy, and per row and alternative its log probability and its class (``None`` without
    alternatives)."""

    log_probs: Tensor
    entropy: Tensor
    top_log_probs: Tensor | None
    top_ids: Tensor | None


def _class_targets(what: str, tl: Tensor, target: Any,
                   ignore_index: int) -> tuple[DeviceArray, int | None]:
    """Class targets of ``tl``'s rows on the device as int64, checked as
    :func:`cross_entropy` checks them: host targets here, device-resident ones by the kernel
    through the returned flag word."""
    dev_t = target.data if isinstance(target, Tensor) else target
    on_device = isinstance(dev_t, DeviceArray)
    t = dev_t if on_device else np.asarray(target)
    if t.dtype.kind not in "iu":
        raise TypeError(f"{what} targets must be integers, got {t.dtype}")
    if tl.shape[:-1] != t.shape:
        raise ValueError(f"logits {tl.shape} and targets {t.shape} are incompatible")
    if on_device:
        if t.dtype != np.int64:
            raise TypeError(f"{what} targets on the device must be int64, got {t.dtype}")
        return t, device.async_error_word(device.ASYNC_CLASS_TARGET)
    flat = np.ascontiguousarray(t.reshape(-1), dtype=np.int64)
    if np.any((flat != ignore_index) & ((flat < 0) | (flat >= tl.shape[-1]))):
        raise IndexError(f"target out of range for {tl.shape[-1]} classes")
    return device.from_numpy(flat), None


class _PartGradients:
    """The gradient of a packed result as the gradients of its parts, by their offsets: the
    engine's sum over the parts' VJPs joins them without device work."""

    __slots__ = ("parts", "shape")

    def __init__(self, shape: tuple[int, ...], parts: dict[int, DeviceArray]) -> None:
        self.shape, self.parts = shape, parts

    def __add__(self, other: _PartGradients) -> _PartGradients:
        parts = dict(self.parts)
        for offset, g in other.parts.items():
            parts[offset] = parts[offset] + g if offset in parts else g
        return _PartGradients(self.shape, parts)

    def pointer(self, offset: int, dtype: np.dtype[Any], keep: list[DeviceArray]) -> int | None:
        """Address of a part's gradient in ``dtype`` (kept alive in ``keep``), None without one."""
        g = self.parts.get(offset)
        if g is None:
            return None
        keep.append(g if g.dtype == dtype else cast_array(g, dtype))
        return keep[-1].ptr


def _part(packed: Tensor, offset: int, shape: tuple[int, ...]) -> Tensor:
    """A contiguous part of a packed result as a view. Its VJP hands the gradient on as that
    part's; the graph VJP puts it into zeros of the packed size."""
    total, count = packed.size, math.prod(shape)

    def backward(g: DeviceArray, need: Need) -> tuple[Any]:
        return (_PartGradients((total,), {offset: g}),)

    def graph(g: Tensor, y: Tensor, need: Need) -> tuple[Tensor]:
        from tensorgrad_b200.ops.shape import _scatter, reshape

        return (_scatter(reshape(g, (count,)), (total,), slice(offset, offset + count)),)

    return make_result(packed.data.flat_view(offset, count, shape), (packed,), backward,
                       "token_log_probs", graph)


@profiled("token_log_probs")
def token_log_probs(logits: Any, targets: Any, *, top_k: int = 0,
                    ignore_index: int = -100) -> TokenLogProbs:
    """The given tokens' log probabilities under ``softmax(logits)``, class axis last, with
    the distribution's entropy and its ``top_k`` likeliest classes (in descending order, equal
    ones by ascending class), all from one pass over the logits.

    Rows whose target is ``ignore_index`` have log probability 0 (their entropy and
    alternatives count). Logits of ``-inf`` close a class: probability 0, nothing added. A row
    without a finite logit, or with a NaN or ``+inf``, gives NaN. Targets are checked as
    :func:`cross_entropy` checks them. Log probabilities, entropy and the alternatives' log
    probabilities are differentiable in the logits (``top_ids`` is a constant choice).
    """
    tl = as_tensor(logits)
    if tl.ndim == 0 or tl.shape[-1] == 0:
        raise ValueError(f"token_log_probs needs a class axis, got logits {tl.shape}")
    lead, classes = tl.shape[:-1], tl.shape[-1]
    if top_k != 0:
        most = min(int(lib.tg_token_log_probs_max_top()), classes)
        if not 0 <= top_k <= most:
            raise ValueError(f"top_k must be in [0, {most}] for {classes} classes, got {top_k}")
    tgt, bad = _class_targets("token_log_probs", tl, targets, ignore_index)
    x = tl.data if tl.dtype.kind == "f" else cast_array(tl.data, np.dtype(np.float64))
    rows = math.prod(lead)
    code = dtype_code(x.dtype)
    es = x.itemsize
    # One buffer: log probabilities, entropies and (row, alternative) log probabilities, which
    # are the result, then the rows' maxima and sums for the VJP.
    size = rows * (2 + top_k)
    whole = device.empty((size + 2 * rows,), x.dtype)
    out, stats = whole.ptr, whole.ptr + size * es
    ids = device.empty((*lead, top_k), np.int64) if top_k else None
    ids_ptr = ids.ptr if ids is not None else None
    check(lib.tg_token_log_probs_forward(
        code, x.ptr, tgt.ptr, stats, out, out + rows * es, out + 2 * rows * es, ids_ptr, rows,
        classes, top_k, ignore_index, bad, device.stream()), "token_log_probs")
    top_ids = Tensor._wrap(ids) if ids is not None else None
    if not (tl.requires_grad and is_grad_enabled()):
        return TokenLogProbs(
            Tensor._wrap(whole.flat_view(0, rows, lead)),
            Tensor._wrap(whole.flat_view(rows, rows, lead)),
            None if ids is None else
            Tensor._wrap(whole.flat_view(2 * rows, rows * top_k, ids.shape)), top_ids)

    def backward(g: Any, need: Need) -> tuple[DeviceArray]:
        # Only the parts' VJPs reach this node.
        keep: list[DeviceArray] = []
        given = [g.pointer(at, x.dtype, keep) for at in (0, rows, 2 * rows)]
        grad = device.empty(tl.shape, x.dtype)
        check(lib.tg_token_log_probs_backward(
            code, x.ptr, tgt.ptr, whole.ptr + size * es, whole.ptr + rows * es, ids_ptr, *given,
            grad.ptr, rows, classes, top_k, ignore_index, device.stream()),
            "token_log_probs backward")
        return (grad if grad.dtype == tl.dtype else cast_array(grad, tl.dtype),)

    def graph(g: Tensor, y: Tensor, need: Need) -> tuple[Tensor | None, ...]:
        return graph_by_composite((tl,), lambda t: _scores_composite(t, tgt, ids, rows, classes,
                                                                     top_k, ignore_index),
                                  g, need)

    packed = make_result(whole.flat_view(0, size), (tl,), backward, "token_log_probs", graph)
    return TokenLogProbs(
        _part(packed, 0, lead), _part(packed, rows, lead),
        None if ids is None else _part(packed, 2 * rows, ids.shape), top_ids)


def _scores_composite(tl: Tensor, tgt: DeviceArray, ids: DeviceArray | None, rows: int,
                      classes: int, top_k: int, ignore_index: int) -> Tensor:
    """The packed result of :func:`token_log_probs` in differentiable ops, with the targets
    and the alternatives found (read back to the host) as constants."""
    from tensorgrad_b200.ops.activation import log_softmax
    from tensorgrad_b200.ops.elementwise import exp, mul, neg
    from tensorgrad_b200.ops.shape import concat, getitem, masked_fill, reshape

    lp = log_softmax(reshape(tl, (rows, classes)), -1)
    # A class without probability is left out of the entropy alone, by p log p = 0; as a target
    # or an alternative its log probability has the gradient of any other's.
    p = exp(lp)
    none = p.numpy() == 0
    p_log_p = mul(masked_fill(p, none, 0.0), masked_fill(lp, none, 0.0))
    t = tgt.numpy().reshape(-1)
    kept = (t != ignore_index) & (t >= 0) & (t < classes)
    at = np.arange(rows)
    given = masked_fill(getitem(lp, (at, np.where(kept, t, 0))), ~kept, 0.0)
    parts = [given, neg(reduce.sum(p_log_p, axis=-1))]
    if ids is not None:
        alt = ids.numpy().reshape(rows, top_k)
        parts.append(reshape(getitem(lp, (at[:, None], alt)), (rows * top_k,)))
    return concat(parts)
