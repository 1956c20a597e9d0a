"""Pre-LN transformer blocks and the GPT language model on the device, with KV-cache
generation (API of the reference's nn/transformer.py:24-220).

The model is a stack of ``x + attn(ln1(x))``, ``x + mlp(ln2(x))`` blocks between token +
position embeddings and a final LayerNorm and vocabulary head, the head sharing the token
embedding's parameter (the engine then sums both gradient contributions into it).
Initialisation is GPT-2's, drawn from the global generator in the reference's order so a
seeded model starts from the reference's weights. Generation keeps per-layer keys and values
on the device (``nn.attention.LayerCache``), so a new token costs one position per layer;
only the last position's logits come back to the host for sampling.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from dataclasses import dataclass
from typing import Any

import numpy as np

from tensorgrad_b200 import device
from tensorgrad_b200._random import get_rng
from tensorgrad_b200.autograd import is_grad_enabled, no_grad
from tensorgrad_b200.nn.attention import LayerCache, MultiHeadAttention
from tensorgrad_b200.nn.layers import (
    GELU, Dropout, Embedding, Int8Linear, LayerNorm, Linear, Sequential,
)
from tensorgrad_b200.nn.module import Module
from tensorgrad_b200.nn.paged import PagedBatch, PagedKVCache, PagedLayer
from tensorgrad_b200.ops.loss import token_log_probs
from tensorgrad_b200.ops.shape import concat
from tensorgrad_b200.tensor import Tensor
from tensorgrad_b200.utils.grad_checkpoint import checkpoint

__all__ = ["GPT", "GPTConfig", "KVCache", "Sampled", "TransformerBlock"]


class TransformerBlock(Module):
    """Pre-LN block: ``x + attn(ln1(x))`` then ``x + mlp(ln2(x))``; the MLP is
    ``Linear(D, r D) -> GELU -> Linear(r D, D) -> Dropout``."""

    def __init__(self, embed_dim: int, num_heads: int, dropout: float = 0.0,
                 mlp_ratio: int = 4) -> None:
        super().__init__()
        hidden = mlp_ratio * embed_dim
        self.ln1 = LayerNorm(embed_dim)
        self.attn = MultiHeadAttention(embed_dim, num_heads, dropout=dropout, causal=True)
        self.ln2 = LayerNorm(embed_dim)
        self.mlp = Sequential(Linear(embed_dim, hidden), GELU(), Linear(hidden, embed_dim),
                              Dropout(dropout))

    def forward(self, x: Tensor, cache: LayerCache | PagedLayer | None = None) -> Tensor:
        x = x + self.attn(self.ln1(x), cache)
        return x + self.mlp(self.ln2(x))


@dataclass
class KVCache:
    """Every layer's cached keys and values for the tokens a :class:`GPT` has processed."""

    layers: list[LayerCache]

    @property
    def length(self) -> int:
        """Positions already cached."""
        return self.layers[0].length if self.layers else 0


@dataclass
class Sampled:
    """One continuation of :meth:`GPT.generate_batch`: the prompt's and the new ids, and the
    new ids' log probabilities under the model (before temperature and top-k)."""

    ids: np.ndarray
    log_probs: np.ndarray


@dataclass(frozen=True)
class GPTConfig:
    """Hyper-parameters of :class:`GPT`."""

    vocab_size: int
    block_size: int = 64
    n_layer: int = 4
    n_head: int = 4
    n_embd: int = 128
    dropout: float = 0.0
    tie_weights: bool = True


_RESIDUAL_OUTPUTS = ("attn.proj", "mlp.2")


class GPT(Module):
    """Decoder-only transformer language model: ids ``(B, T)`` to logits ``(B, T, V)``.

    With :attr:`gradient_checkpointing` set, a training forward pass keeps only the residual
    stream between blocks and recomputes each block in the backward pass
    (``tensorgrad_b200.utils.checkpoint``; the reference's nn/transformer.py:155-159)."""

    gradient_checkpointing: bool

    def __init__(self, config: GPTConfig) -> None:
        super().__init__()
        self.config = config
        self.tok_emb = Embedding(config.vocab_size, config.n_embd)
        self.pos_emb = Embedding(config.block_size, config.n_embd)
        self.drop = Dropout(config.dropout)
        self.blocks = Sequential(*[TransformerBlock(config.n_embd, config.n_head, config.dropout)
                                   for _ in range(config.n_layer)])
        self.ln_f = LayerNorm(config.n_embd)
        self.head = Linear(config.n_embd, config.vocab_size, bias=False)
        self._gpt2_init()
        if config.tie_weights:
            self.head.weight = self.tok_emb.weight
        self.gradient_checkpointing = False

    def _gpt2_init(self) -> None:
        """N(0, 0.02) for every linear weight and embedding, N(0, 0.02 / sqrt(2 L)) for the
        projections that write into the residual stream, zero biases; drawn module by module
        in traversal order."""
        rng = get_rng()
        narrow = 0.02 / math.sqrt(2 * self.config.n_layer)
        for name, module in self.named_modules():
            if not isinstance(module, Linear | Embedding):
                continue
            std = narrow if (isinstance(module, Linear) and name.endswith(_RESIDUAL_OUTPUTS)) \
                else 0.02
            module.weight.data[...] = rng.normal(0.0, std, size=module.weight.shape)
            bias = getattr(module, "bias", None)
            if bias is not None:
                bias.data.fill_(0.0)

    def quantize_int8(self, head: bool = False) -> GPT:
        """Turn this model into one for inference whose blocks' linear layers (and with
        ``head`` the vocabulary head) hold their weights in 8-bit integers
        (:class:`Int8Linear`). The other parameters stop requiring gradients; a tied
        embedding keeps its floating table."""
        for block in self.blocks:
            for parent, name in ((block.attn, "qkv"), (block.attn, "proj"), (block.mlp, "0"),
                                 (block.mlp, "2")):
                layer = getattr(parent, name)
                if isinstance(layer, Linear):
                    setattr(parent, name, Int8Linear(layer))
        if head and isinstance(self.head, Linear):
            self.head = Int8Linear(self.head)
        for p in self.parameters():
            p.requires_grad = False
        return self.eval()

    # ------------------------------------------------------------------ forward
    def forward(self, idx: Any, cache: KVCache | PagedBatch | None = None) -> Tensor:
        """Logits for token ids ``(B, T)``; with a ``cache``, ids continue the cached ones
        (positions from ``cache.length``, or each row's own length in a
        ``PagedKVCache.batch``; inference only, no graph). Host ids are checked
        on the host; ids in a device tensor stay on the device (checked there)."""
        tokens = idx if isinstance(idx, Tensor) else np.asarray(idx)
        if tokens.ndim != 2:
            raise ValueError(f"expected (B, T) token ids, got shape {tokens.shape}")
        if isinstance(cache, PagedBatch):
            return self._forward_paged(tokens, cache)
        start = cache.length if cache is not None else 0
        t = tokens.shape[1]
        if start + t > self.config.block_size:
            raise ValueError(f"sequence length {start + t} exceeds block_size "
                             f"{self.config.block_size}")
        if cache is None:
            x = self.drop(self.tok_emb(tokens) + self.pos_emb(_positions(0, t)))
            recompute = self.gradient_checkpointing and is_grad_enabled()
            for block in self.blocks:
                x = checkpoint(block, x) if recompute else block(x)
            return self.head(self.ln_f(x))
        if self.training:
            raise ValueError("a KV cache is for inference: call eval() first")
        with no_grad():
            x = self.tok_emb(tokens) + self.pos_emb(_positions(start, t))
            for block, layer in zip(self.blocks, cache.layers, strict=True):
                x = block(x, layer)
            return self.head(self.ln_f(x))

    def _forward_paged(self, tokens: Any, rows: PagedBatch) -> Tensor:
        b, t = tokens.shape
        starts = rows.lengths
        if b != len(starts):
            raise ValueError(f"{b} rows of ids for {len(starts)} sequences")
        if t == 0:
            raise ValueError("a step needs at least one token")
        if int(starts.max()) + t > self.config.block_size:
            raise ValueError(f"sequence length {int(starts.max()) + t} exceeds block_size "
                             f"{self.config.block_size}")
        if self.training:
            raise ValueError("a KV cache is for inference: call eval() first")
        rows.check_model(len(self.blocks), self.blocks[0].attn if len(self.blocks) else None,
                         self.tok_emb.weight.dtype)
        with no_grad():
            steps = rows.begin(t)
            x = self.tok_emb(tokens) + self.pos_emb(starts[:, None] + np.arange(t))
            for block, layer in zip(self.blocks, steps, strict=True):
                x = block(x, layer)
            logits = self.head(self.ln_f(x))
        rows.commit(t)
        return logits

    # ------------------------------------------------------------------ generation
    def make_cache(self, batch_size: int) -> KVCache:
        """Empty per-layer device caches for ``batch_size`` sequences of ``block_size``."""
        dt = self.tok_emb.weight.dtype
        return KVCache([LayerCache.empty(batch_size, blk.attn.num_heads, self.config.block_size,
                                         blk.attn.head_dim, dt) for blk in self.blocks])

    def make_paged_cache(self, num_pages: int, page_size: int = 16) -> PagedKVCache:
        """An empty cache of ``num_pages`` pages of ``page_size`` positions for this model's
        layers, to be shared by any number of sequences."""
        attn = self.blocks[0].attn
        return PagedKVCache(self.config.n_layer, attn.num_heads, attn.head_dim, num_pages,
                            page_size, self.tok_emb.weight.dtype)

    def generate_batch(self, prompts: Sequence[Any], max_new_tokens: int, *, samples: int = 1,
                       temperature: float = 1.0, top_k: int | None = None,
                       rng: np.random.Generator | None = None,
                       page_size: int = 16) -> list[list[Sampled]]:
        """``samples`` continuations of each prompt (1-D ids of any lengths, each at least
        one) by ``max_new_tokens`` sampled tokens, all in one batch over a paged cache: a
        prompt is encoded once and forked, every step then costs one position per
        continuation. Prompts and new tokens have to fit in ``block_size``. Sampling is
        :meth:`generate`'s, row by row in the order of the result."""
        if temperature <= 0:
            raise ValueError("temperature must be positive")
        if samples < 1 or max_new_tokens < 0:
            raise ValueError(f"cannot draw {samples} samples of {max_new_tokens} tokens")
        if page_size < 1:
            raise ValueError(f"page_size must be positive, got {page_size}")
        texts = [np.asarray(p, dtype=np.int64) for p in prompts]
        for p in texts:
            if p.ndim != 1 or p.size == 0:
                raise ValueError(f"expected prompts of at least one id, got shape {p.shape}")
            if p.size + max_new_tokens > self.config.block_size:
                raise ValueError(f"sequence length {p.size + max_new_tokens} exceeds block_size "
                                 f"{self.config.block_size}")
        if not texts:
            return []
        gen = rng or get_rng()
        was_training = self.training
        self.eval()
        most = sum(-(-(p.size + max_new_tokens) // page_size) for p in texts) * samples
        ids = [p for p in texts for _ in range(samples)]
        scores: list[list[np.ndarray]] = [[] for _ in ids]
        try:
            cache = self.make_paged_cache(most, page_size)
            rows: list[int] = []
            firsts = []
            for p in texts if max_new_tokens else ():
                seq = cache.add()
                firsts.append(self(p[None], cache=cache.batch([seq]))[:, -1])
                rows += [seq, *(cache.fork(seq) for _ in range(samples - 1))]
            logits = concat([f for f in firsts for _ in range(samples)]) if firsts else None
            for step in range(max_new_tokens):
                new = _sample(logits.numpy().astype(np.float64) / temperature, top_k, gen)
                found = token_log_probs(logits, new).log_probs.numpy()
                for i, token in enumerate(new):
                    ids[i] = np.append(ids[i], token)
                    scores[i].append(found[i])
                if step + 1 < max_new_tokens:
                    logits = self(new[:, None], cache=cache.batch(rows))[:, -1]
        finally:
            self.train(was_training)
        out = [Sampled(i, np.array(s, dtype=self.tok_emb.weight.dtype))
               for i, s in zip(ids, scores, strict=True)]
        return [out[k:k + samples] for k in range(0, len(out), samples)]

    def generate(self, idx: Any, max_new_tokens: int, *, temperature: float = 1.0,
                 top_k: int | None = None, rng: np.random.Generator | None = None,
                 use_cache: bool = True) -> np.ndarray:
        """Extend ids ``(B, T)`` by ``max_new_tokens`` sampled tokens (evaluation mode, no
        graph). The context is the last ``block_size`` tokens; ``top_k`` keeps the k most
        likely tokens; ``rng`` defaults to the global generator. With ``use_cache`` each new
        token is one position per layer against the device KV cache while the sequence fits
        in ``block_size``; once the window slides, the (absolute) positions shift and the
        window is encoded afresh, so both settings give the same tokens."""
        if temperature <= 0:
            raise ValueError("temperature must be positive")
        gen = rng or get_rng()
        was_training = self.training
        self.eval()
        out = np.asarray(idx, dtype=np.int64)
        window = self.config.block_size
        try:
            with no_grad():
                cache: KVCache | None = None
                for _ in range(max_new_tokens):
                    if not use_cache:
                        logits = self(out[:, -window:])
                    elif cache is not None and cache.length == out.shape[1] - 1:
                        logits = self(out[:, -1:], cache=cache)
                    else:
                        cache = self.make_cache(len(out))
                        logits = self(out[:, -window:], cache=cache)
                    if out.shape[1] >= window:
                        cache = None
                    last = _last_position(logits).astype(np.float64) / temperature
                    out = np.concatenate([out, _sample(last, top_k, gen)[:, None]], axis=1)
        finally:
            self.train(was_training)
        return out


def _last_position(logits: Tensor) -> np.ndarray:
    """The last position's logits ``(B, V)`` on the host (one small copy)."""
    b, t, v = logits.shape
    return logits.data.flat_view(0, b * t * v, (b, t, v)).numpy()[:, -1, :]


def _sample(logits: np.ndarray, top_k: int | None, gen: np.random.Generator) -> np.ndarray:
    """One token per row from ``softmax(logits)`` after an optional top-k cut, drawn as the
    reference does (a max-shifted softmax in float64, then ``Generator.choice``)."""
    if top_k is not None:
        kth = np.sort(logits, axis=-1)[:, -min(top_k, logits.shape[-1])]
        logits = np.where(logits < kth[:, None], -np.inf, logits)
    peak = logits.max(axis=-1, keepdims=True)
    e = np.exp(logits - np.where(np.isfinite(peak), peak, 0))
    probs = e / e.sum(axis=-1, keepdims=True)
    return np.array([gen.choice(probs.shape[-1], p=row) for row in probs])


_POSITIONS: dict[tuple[int, int, str], Tensor] = {}


def _positions(start: int, t: int) -> Tensor:
    """Positions ``start .. start + t - 1`` as a device tensor, uploaded once per range."""
    key = (start, t, str(device.current_device()))
    p = _POSITIONS.get(key)
    if p is None:
        if len(_POSITIONS) > 4096:
            _POSITIONS.clear()
        p = _POSITIONS[key] = Tensor(np.arange(start, start + t, dtype=np.int64))
    return p
