"""tensorgrad_b200: tensorgrad's training step on B200 GPUs.

The top-level namespace mirrors ``tensorgrad`` (the reference): the :class:`Tensor` type,
grad-mode switches, factories and the differentiable ops; ``nn``, ``optim`` and ``autograd``
are the same modules. Tensors live in device memory and every op runs hand-written sm_100a
kernels from ``libtgb200.so`` (C ABI in ``include/tgb200.h``); there is no CPU fallback.
"""

from tensorgrad_b200 import autograd, profiler
from tensorgrad_b200._random import get_rng, manual_seed
from tensorgrad_b200.autograd import enable_grad, is_grad_enabled, no_grad
from tensorgrad_b200.device import DeviceArray, set_device, synchronize
from tensorgrad_b200.ops import (
    Int8Weight, add, append_pages, binary_cross_entropy_with_logits, broadcast_to, concat,
    conv2d, copy_pages, cross_entropy, div, dropout, embedding, exp, flatten, gather_pages,
    gelu, int8_linear, layer_norm, linear, log, log_softmax, logsumexp, masked_fill, matmul,
    max, max_pool2d, mean, min, mse_loss, mul, neg, paged_attention, permute, pow,
    quantize_int8, relu, reshape, sigmoid, softmax, sqrt, squeeze, stack, sub, sum, tanh,
    token_log_probs, transpose, unsqueeze, var, where,
)
from tensorgrad_b200.tensor import (
    Tensor, arange, full, get_default_dtype, ones, ones_like, rand, randn, set_default_dtype,
    tensor, zeros, zeros_like,
)

from tensorgrad_b200 import func, nn, optim, utils, viz  # noqa: E402  (after the ops they use)

__version__ = "0.1.0"


def _lib_launches() -> int:
    """Kernels launched by libtgb200.so in this process so far."""
    from tensorgrad_b200._lib import lib

    return int(lib.tg_launch_count())

__all__ = [
    "DeviceArray", "Int8Weight", "Tensor", "__version__", "add", "append_pages", "arange",
    "autograd", "binary_cross_entropy_with_logits", "broadcast_to", "concat", "conv2d",
    "copy_pages", "cross_entropy", "div", "dropout", "embedding", "enable_grad", "exp",
    "flatten", "full", "func", "gather_pages", "gelu", "get_default_dtype", "get_rng",
    "int8_linear", "is_grad_enabled", "layer_norm", "linear", "log", "log_softmax",
    "logsumexp", "manual_seed", "masked_fill", "matmul", "max", "max_pool2d", "mean", "min",
    "mse_loss", "mul", "neg", "nn", "no_grad", "ones", "ones_like", "optim",
    "paged_attention", "permute", "pow", "profiler", "quantize_int8", "rand", "randn", "relu",
    "reshape", "set_default_dtype", "set_device", "sigmoid", "softmax", "sqrt", "squeeze",
    "stack", "sub", "sum", "synchronize", "tanh", "tensor", "token_log_probs", "transpose",
    "unsqueeze", "utils", "var", "viz", "where", "zeros", "zeros_like",
]
