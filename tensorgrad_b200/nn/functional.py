"""Functional interface (``import tensorgrad_b200.nn.functional as F``), as the reference's."""

from tensorgrad_b200.ops import (  # noqa: F401
    batch_norm, binary_cross_entropy_with_logits, conv2d, cross_entropy, dropout, embedding,
    gelu, gru, int8_linear, layer_norm, linear, log_softmax, lstm, max_pool2d, mse_loss, relu, rnn, sigmoid,
    softmax, tanh, token_log_probs,
)
from tensorgrad_b200.ops.attention import (  # noqa: F401
    packed_self_attention, scaled_dot_product_attention,
)
from tensorgrad_b200.ops.paged import paged_attention  # noqa: F401
