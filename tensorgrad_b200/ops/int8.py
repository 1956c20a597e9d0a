"""Linear layers in 8-bit integers for inference (no counterpart in the reference; the form of
ops/layers.py:22-62 that serves a trained model).

The weight is quantised once, each output channel by its own scale; the input is quantised in
the call, each token (row) by its own: ``scale = max|x| * (1 / 127)`` and the nearest integers to
``x / scale``. The products are summed exactly in 32-bit integers and scaled once.
"""

from __future__ import annotations

from typing import Any

import numpy as np

from tensorgrad_b200 import device
from tensorgrad_b200._lib import check, lib
from tensorgrad_b200.autograd import is_grad_enabled
from tensorgrad_b200.device import DeviceArray, dtype_code
from tensorgrad_b200.ops._util import as_tensor
from tensorgrad_b200.ops.elementwise import cast_array
from tensorgrad_b200.profiler import profiled
from tensorgrad_b200.tensor import Tensor

__all__ = ["Int8Weight", "int8_linear", "quantize_int8"]

_ROW = 16  # integer rows start on 16-byte boundaries


def _padded(inner: int) -> int:
    return -(-inner // _ROW) * _ROW


def _device_array(x: Any) -> DeviceArray:
    if isinstance(x, Tensor):
        return x.data
    return x if isinstance(x, DeviceArray) else device.from_numpy(np.asarray(x))


class Int8Weight:
    """A linear layer's weight as integers ``q`` ``(out_features, row)`` and a scale for each
    output channel: the weight is ``q[:, :in_features] * scale[:, None]``. Rows are a multiple of
    16 bytes long; what is behind ``in_features`` does not count. Integers in other rows are
    laid out anew; :meth:`quantize` makes one from a floating weight."""

    __slots__ = ("in_features", "q", "scale")

    def __init__(self, q: Any, scale: Any, in_features: int | None = None) -> None:
        if isinstance(q, np.ndarray) and q.ndim == 2 and q.dtype == np.int8:
            inner = q.shape[1] if in_features is None else in_features
            if 0 < inner <= q.shape[1]:  # a host weight is laid out before it goes up
                rows = np.zeros((q.shape[0], _padded(inner)), dtype=np.int8)
                rows[:, :inner] = q[:, :inner]
                q, in_features = rows, inner
        a, s = _device_array(q), _device_array(scale)
        if a.dtype != np.int8 or len(a.shape) != 2:
            raise TypeError(f"expected int8 integers (out_features, row), got {a.dtype} "
                            f"{tuple(a.shape)}")
        inner = a.shape[1] if in_features is None else in_features
        if not 0 < inner <= a.shape[1]:
            raise ValueError(f"in_features must be in [1, {a.shape[1]}], got {inner}")
        if s.dtype.kind != "f" or tuple(s.shape) != (a.shape[0],):
            raise ValueError(f"expected {a.shape[0]} floating scales, got {s.dtype} "
                             f"{tuple(s.shape)}")
        if a.shape[1] % _ROW or a.ptr % _ROW:
            host = a.numpy()
            rows = np.zeros((a.shape[0], _padded(inner)), dtype=np.int8)
            rows[:, :inner] = host[:, :inner]
            a = device.from_numpy(rows)
        self.q, self.scale, self.in_features = a, s, inner

    @property
    def out_features(self) -> int:
        return self.q.shape[0]

    @classmethod
    def quantize(cls, weight: Any) -> Int8Weight:
        """The integers of a floating weight ``(out_features, in_features)``."""
        w = as_tensor(weight)
        if w.ndim != 2 or w.shape[1] == 0:
            raise ValueError(f"expected a weight (out_features, in_features), got {w.shape}")
        q, scale = _quantize_rows(w.data, _padded(w.shape[1]))
        return cls(q, scale, w.shape[1])

    def __repr__(self) -> str:
        return f"Int8Weight({self.out_features}, {self.in_features}, scale {self.scale.dtype})"


def _quantize_rows(x: DeviceArray, ld: int) -> tuple[DeviceArray, DeviceArray]:
    code = dtype_code(x.dtype)
    inner = x.shape[-1]
    rows = x.size // inner
    q, scale = device.empty((rows, ld), np.int8), device.empty((rows,), x.dtype)
    check(lib.tg_int8_quantize_rows(code, x.ptr, rows, inner, q.ptr, ld, scale.ptr,
                                    device.stream()), "quantize_int8")
    return q, scale


@profiled("quantize_int8")
def quantize_int8(x: Any) -> tuple[Tensor, Tensor]:
    """``x`` over its last axis as 8-bit integers of ``x``'s shape and one scale per row
    (``x.shape[:-1]``): ``scale = max|row| * (1 / 127)``, the factor rounded to the type, and
    the nearest integers to ``row / scale`` rounded to the type, halves to even. A row of zeros
    has scale 0; a row with a NaN or an infinity has scale NaN and integers 0. Both results are
    constants: no gradient reaches ``x`` through them, whether or not it requires one."""
    tx = as_tensor(x)
    if tx.ndim == 0 or tx.shape[-1] == 0:
        raise ValueError(f"quantize_int8 needs a last axis with values, got {tx.shape}")
    dtype_code(tx.dtype)
    q, scale = _quantize_rows(tx.data, tx.shape[-1])
    return Tensor._wrap(q.reshape(tx.shape)), Tensor._wrap(scale.reshape(tx.shape[:-1]))


@profiled("int8_linear")
def int8_linear(x: Any, weight: Int8Weight, bias: Any = None) -> Tensor:
    """``x @ W.T + bias`` over flattened leading axes with ``W`` in 8-bit integers and ``x``
    quantised row by row in the call (see :func:`quantize_int8`); the result has ``x``'s
    floating type. Inference only."""
    tx = as_tensor(x)
    if not isinstance(weight, Int8Weight):
        raise TypeError(f"int8_linear takes an Int8Weight, got {type(weight).__name__}")
    if tx.ndim == 0 or tx.shape[-1] != weight.in_features:
        raise ValueError(f"int8_linear: input {tx.shape} does not match weight "
                         f"{(weight.out_features, weight.in_features)}")
    code = dtype_code(tx.dtype)
    tb = None if bias is None else as_tensor(bias)
    if tb is not None and tb.shape != (weight.out_features,):
        raise ValueError(f"int8_linear: bias {tb.shape} for {weight.out_features} channels")
    if is_grad_enabled() and (tx.requires_grad or (tb is not None and tb.requires_grad)):
        raise ValueError("int8_linear is for inference: use no_grad() or detach its inputs")
    x_, inner, outer = tx.data, weight.in_features, weight.out_features
    scale = weight.scale if weight.scale.dtype == x_.dtype else cast_array(weight.scale, x_.dtype)
    b = None
    if tb is not None:
        b = tb.data if tb.dtype == x_.dtype else cast_array(tb.data, x_.dtype)
    rows = x_.size // inner
    y = device.empty((*tx.shape[:-1], outer), x_.dtype)
    nbytes = lib.tg_int8_linear_scratch_bytes(code, rows, inner, outer)
    scratch = device.scratch(nbytes) if nbytes > 16 else None
    check(lib.tg_int8_linear(code, x_.ptr, rows, inner, weight.q.ptr, weight.q.shape[1],
                             scale.ptr, None if b is None else b.ptr, y.ptr, outer,
                             None if scratch is None else scratch.ptr, device.stream()),
          "int8_linear")
    return Tensor._wrap(y)
