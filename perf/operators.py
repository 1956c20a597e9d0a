"""The serving operators of the GPT path, with their cases: log probabilities of given tokens
(with the entropy and the likeliest alternatives, forward and backward), attention of one new
token over a paged key-value cache, the operations on the cache's pages, and the linear layer
in 8-bit integers with a scale for each token and each channel.

``own`` selects what :func:`run` computes with: false, the operators' plain forms in elementary
torch operations; true, the calls of ``tensorgrad_b200``. Inputs live in torch's memory; the
calls view them in place and their results are viewed back, nothing is copied on the way.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

IGNORE = -100
_TYPES = {"f32": torch.float32, "f64": torch.float64}


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # One sampling step of 16 sequences over GPT-2's padded vocabulary: the chosen tokens'
        # log probabilities, the entropy and the 20 likeliest tokens.
        dict(name="score_step", op="score", rows=16, classes=50304, top_k=20, backward=False, type="f32"),
        # A training step on 8 sequences of 1024 tokens: log probabilities and an entropy bonus,
        # with the gradient of the logits.
        dict(name="score_train", op="score", rows=8192, classes=50304, top_k=0, backward=True, type="f32"),
        # An odd vocabulary in the float64 mode, with gradients through the alternatives too.
        dict(name="score_odd_f64", op="score", rows=257, classes=32003, top_k=5, backward=True, type="f64"),
        # One sequence of a 12-head model, somewhere in its 1024 positions: latency.
        dict(name="decode_one", op="decode", batch=1, kv_heads=12, group=1, width=64, page=16, longest=1024, type="f32"),
        # A serving batch of the same model, sequences of every length.
        dict(name="decode_batch", op="decode", batch=64, kv_heads=12, group=1, width=64, page=16, longest=1024, type="f32"),
        # Few long contexts, four query heads to a key head.
        dict(name="decode_long", op="decode", batch=4, kv_heads=8, group=4, width=128, page=32, longest=65536, type="f32"),
        # Odd head width and pages of 5 positions in the float64 mode.
        dict(name="decode_odd_f64", op="decode", batch=9, kv_heads=5, group=2, width=40, page=5, longest=700, type="f64"),
        # Compaction of a 12-layer cache: 1024 pages move to the front of both pools.
        dict(name="compact_pages", op="copy", layers=12, kv_heads=12, width=64, page=16, pool=2600, pairs=1024, type="f32"),
        # One layer of a decode step of 256 sequences writes the new keys and values.
        dict(name="append_step", op="append", batch=256, tokens=1, kv_heads=12, width=64, page=16, longest=1024, type="f32"),
        # The fused query/key/value projection of a 768-wide model for one new token.
        dict(name="int8_token", op="int8", rows=1, inner=768, outer=2304, bias=True, type="f32"),
        # A ragged batch of prompts through an odd layer.
        dict(name="int8_odd", op="int8", rows=333, inner=1001, outer=1999, bias=True, type="f32"),
        # 8192 prompt tokens through a wide layer: the tensor cores' case.
        dict(name="int8_prompt", op="int8", rows=8192, inner=4096, outer=4096, bias=False, type="f32"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(("score", "score", "decode", "decode", "decode", "copy", "append", "gather", "int8", "int8"))
    kind = "f64" if rng.random() < 0.2 else "f32"
    if op == "score":
        top_k = rng.choice((0, 0, 1, 5, 20, rng.randint(1, 100)))
        cells = 1e8 if top_k or kind == "f64" else 4e8
        classes = _spread(rng, 17, 60000)
        rows = _spread(rng, 1, int(min(8192, cells // classes)))
        return dict(op=op, rows=rows, classes=classes, top_k=min(top_k, classes), backward=rng.random() < 0.5, type=kind)
    if op == "int8":
        rows, inner = _spread(rng, 1, 8192), _spread(rng, 16, 8192)
        outer = _spread(rng, 8, int(min(50304, 6e7 // rows, 1.3e11 // (rows * inner))))
        if kind == "f64":
            rows = min(rows, 512)
        return dict(op=op, rows=rows, inner=inner, outer=outer, bias=rng.random() < 0.7, type=kind)
    width = rng.choice((16, 32, 40, 64, 64, 64, 80, 128, 128, rng.randint(1, 256)))
    page = rng.choice((1, 5, 8, 16, 16, 32, 64, rng.randint(2, 100)))
    heads = rng.choice((1, 2, 3, 4, 8, 12))
    if op == "copy":
        layers = rng.choice((1, 2, 6, 12))
        most = int(min(1024, 1.2e9 // (layers * heads * width * page * 16)))
        pairs = _spread(rng, 1, max(1, most))
        return dict(op=op, layers=layers, kv_heads=heads, width=width, page=page, pool=2 * pairs + rng.randint(0, 50), pairs=pairs, type=kind)
    per = heads * width * (16 if kind == "f64" else 8)
    cells = 5e8 / per if op == "gather" else 1.5e9 / per
    batch = _spread(rng, 1, 128)
    longest = _spread(rng, 1, int(min(65536, max(1, cells // batch))))
    if op == "decode":
        return dict(op=op, batch=batch, kv_heads=heads, group=rng.choice((1, 1, 2, 3, 4, 8)), width=width, page=page, longest=longest, type=kind)
    if op == "gather":
        return dict(op=op, batch=batch, kv_heads=heads, width=width, page=page, longest=longest, type=kind)
    return dict(op=op, batch=batch, tokens=min(longest, _spread(rng, 1, 512)), kv_heads=heads, width=width, page=page, longest=longest, type=kind)


def _size(case):
    return 8 if case["type"] == "f64" else 4


def work(case):
    es, op = _size(case), case["op"]
    if op == "score":
        cells, k = case["rows"] * case["classes"], case["top_k"]
        small = case["rows"] * (8 + 2 * es + k * (es + 8))
        more = cells * es + case["rows"] * (2 + k) * es if case["backward"] else 0
        return {"bytes": cells * es + small + more, "flops": cells * (10 if case["backward"] else 5)}
    if op == "int8":
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"bytes": m * k * es + n * k + n * es * (2 if case["bias"] else 1) + m * n * es, "flops": 2 * m * n * k}
    slot = case["kv_heads"] * case["width"] * 2 * es  # one position's keys and values
    if op == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["page"] * slot + 16 * case["pairs"], "flops": 0}
    if op == "append":
        return {"bytes": 2 * case["batch"] * case["tokens"] * slot + 16 * case["batch"], "flops": 0}
    held = _held(case)
    if op == "gather":
        return {"bytes": (held + case["batch"] * case["longest"]) * slot, "flops": 0}
    heads = case["kv_heads"] * case["group"]
    return {"bytes": held * slot + 2 * case["batch"] * heads * case["width"] * es, "flops": 4 * held * heads * case["width"]}


def _held(case):
    """Positions in the cache, over all sequences, as :func:`_lengths` spreads them."""
    return int(sum(_lengths(case)))


def _lengths(case):
    """The sequences' lengths: one as long as the case allows, the others spread down to a
    quarter of it, and in larger batches one that holds nothing yet."""
    b, longest = case["batch"], case["longest"]
    out = [max(1, longest - (3 * longest * i) // (4 * b)) for i in range(b)]
    if b >= 8:
        out[b // 2] = 0
    return out


# ---------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = np.random.default_rng(int(seed))
    dt, op = _TYPES[case["type"]], case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dt)

    s = SimpleNamespace(case=dict(case), op=op)
    if op == "score":
        rows, classes = case["rows"], case["classes"]
        s.logits = normal(rows, classes).mul_(3.0)
        # A trained model's logits have a few clear favourites; a padded vocabulary's last
        # entries are closed.
        liked = torch.randint(classes, (rows, 4), generator=g, device="cuda")
        s.logits.scatter_add_(1, liked, normal(rows, 4).abs_().mul_(4.0))
        closed = min(classes // 200, 64)
        s.logits[:, classes - closed:] = float("-inf")
        s.targets = torch.randint(classes - closed, (rows,), generator=g, device="cuda")
        s.targets[torch.rand(rows, generator=g, device="cuda") < 0.1] = IGNORE
        s.g_log, s.g_ent, s.g_top = normal(rows), normal(rows), normal(rows, max(case["top_k"], 1))
    elif op == "int8":
        m, k, n = case["rows"], case["inner"], case["outer"]
        s.x = normal(m, k)
        s.x[:, torch.randint(k, (max(1, k // 100),), generator=g, device="cuda")] *= 8.0  # outlying channels
        w = normal(n, k).mul_(k ** -0.5)
        s.scale = w.abs().amax(1) / 127
        # A program's weights are quantised once and kept with rows of a multiple of 16 bytes.
        s.weight = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
        s.weight[:, :k] = torch.round(w / s.scale[:, None]).clamp_(-127, 127).to(torch.int8)
        s.bias = normal(n) if case["bias"] else None
    elif op == "copy":
        shape = (case["layers"], case["pool"], case["kv_heads"], case["page"], case["width"])
        s.keys, s.values = normal(*shape), normal(*shape)
        order = host.permutation(case["pool"])[:2 * case["pairs"]]
        s.dst, s.src = np.sort(order[:case["pairs"]]), order[case["pairs"]:].copy()
    else:
        b, h, d, size = case["batch"], case["kv_heads"], case["width"], case["page"]
        lengths = host.permutation(np.asarray(_lengths(case), dtype=np.int64))
        per = -(-case["longest"] // size)
        pool = b * per + 3
        ids = host.permutation(pool)[:b * per].reshape(b, per)
        s.pages = torch.from_numpy(ids.astype(np.int64)).cuda()
        s.keys, s.values = normal(pool, h, size, d), normal(pool, h, size, d)
        if op == "append":
            lengths = np.minimum(lengths, case["longest"] - case["tokens"])
            s.k, s.v = normal(b, h, case["tokens"], d), normal(b, h, case["tokens"], d)
        s.lengths = torch.from_numpy(lengths).cuda()
        s.longest = case["longest"]
        if op == "decode":
            s.q = normal(b, h * case["group"], d)
    return s


# ---------------------------------------------------------------------- one pass
def run(s):
    return globals()[("own_" if own else "plain_") + s.op](s)


def plain_score(s):
    x, k = s.logits, s.case["top_k"]
    m = x.amax(1, keepdim=True)
    z = x - m
    e = z.exp()
    total = e.sum(1, keepdim=True)
    ls = total.log()
    z = torch.where(e > 0, z, 0.0)
    p = e / total
    ent = ls - (p * z).sum(1, keepdim=True)
    kept = s.targets != IGNORE
    at = torch.where(kept, s.targets, 0)[:, None]
    out = {"log_probs": torch.where(kept, (x.gather(1, at) - m - ls)[:, 0], 0.0), "entropy": ent[:, 0]}
    if k:
        best, ids = x.sort(dim=1, descending=True, stable=True)
        out["top_log_probs"], out["top_ids"] = best[:, :k] - m - ls, ids[:, :k].contiguous()
    if s.case["backward"]:
        pull = (s.g_log * kept)[:, None]
        push = pull + s.g_top[:, :k].sum(1, keepdim=True) if k else pull
        grad = -p * (push + s.g_ent[:, None] * (z - ls + ent))
        grad.scatter_add_(1, at, pull)
        if k:
            grad.scatter_add_(1, out["top_ids"], s.g_top[:, :k])
        out["grad"] = grad
    return out


def plain_decode(s):
    c = s.case
    b, h, n, d, size = c["batch"], c["kv_heads"], c["group"], c["width"], c["page"]
    per = s.pages.shape[1]
    keys = s.keys[s.pages].permute(0, 2, 1, 3, 4).reshape(b, h, per * size, d)
    scores = s.q.view(b, h, n, d) @ keys.transpose(2, 3) * d ** -0.5
    del keys
    seen = (torch.arange(per * size, device="cuda") < s.lengths[:, None])[:, None, None]
    scores = torch.where(seen, scores, float("-inf"))
    m = scores.amax(3, keepdim=True)
    e = torch.where(seen, (scores - m).exp(), 0.0)
    values = s.values[s.pages].permute(0, 2, 1, 3, 4).reshape(b, h, per * size, d)
    total = e.sum(3, keepdim=True)
    out = torch.where(total > 0, (e @ values) / total, 0.0)
    return {"out": out.reshape(b, h * n, d)}


def plain_copy(s):
    src, dst = torch.from_numpy(s.src).cuda(), torch.from_numpy(s.dst).cuda()
    s.keys[:, dst] = s.keys[:, src]
    s.values[:, dst] = s.values[:, src]
    return {"keys": s.keys, "values": s.values}


def plain_append(s):
    size = s.case["page"]
    at = s.lengths[:, None] + torch.arange(s.case["tokens"], device="cuda")
    page, slot = s.pages.gather(1, at // size), at % size
    s.keys[page, :, slot] = s.k.transpose(1, 2)
    s.values[page, :, slot] = s.v.transpose(1, 2)
    return {"keys": s.keys, "values": s.values}


def plain_gather(s):
    b, h, d = s.case["batch"], s.case["kv_heads"], s.case["width"]
    seen = (torch.arange(s.longest, device="cuda") < s.lengths[:, None])[:, None, :, None]
    keys = s.keys[s.pages].permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)[:, :, :s.longest]
    values = s.values[s.pages].permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)[:, :, :s.longest]
    return {"keys": torch.where(seen, keys, 0.0), "values": torch.where(seen, values, 0.0)}


def plain_int8(s):
    scale = s.x.abs().amax(1, keepdim=True) / 127
    q = torch.where(scale > 0, torch.round(s.x / scale), 0.0).clamp_(-127, 127)
    y = (q @ s.weight[:, :s.x.shape[1]].to(q.dtype).T) * (scale * s.scale)
    return {"out": y if s.bias is None else y + s.bias}


# ---------------------------------------------------------------------- the framework's calls
_NP = {torch.float32: np.dtype(np.float32), torch.float64: np.dtype(np.float64),
       torch.int64: np.dtype(np.int64), torch.int8: np.dtype(np.int8)}


def _array(t):
    """A torch tensor's memory as a device array of the framework."""
    from tensorgrad_b200 import DeviceArray

    return DeviceArray(SimpleNamespace(ptr=t.data_ptr(), device=t.device.index, held=t), 0, tuple(t.shape), _NP[t.dtype])


def _tensor(t):
    from tensorgrad_b200 import Tensor

    return Tensor._wrap(_array(t))


class _View:
    def __init__(self, a):
        self.held = a
        self.__cuda_array_interface__ = {"shape": a.shape, "typestr": a.dtype.str, "data": (a.ptr, False), "version": 3}


def _torch(t):
    """A result of the framework as a torch tensor on the same memory."""
    return torch.as_tensor(_View(t.data), device="cuda")


def own_score(s):
    import tensorgrad_b200 as tg
    from tensorgrad_b200.ops._util import make_result

    x, k, arrived = _tensor(s.logits), s.case["top_k"], []
    if s.case["backward"]:
        # The logits are a layer's output: their gradient arrives at that layer's VJP.
        leaf = _tensor(s.g_log)
        leaf.requires_grad = True
        x = make_result(x.data, (leaf,), lambda g, need: (arrived.append(g),), "head")
    got = tg.token_log_probs(x, _tensor(s.targets), top_k=k, ignore_index=IGNORE)
    out = {"log_probs": _torch(got.log_probs), "entropy": _torch(got.entropy)}
    if k:
        out["top_log_probs"], out["top_ids"] = _torch(got.top_log_probs), _torch(got.top_ids)
    if s.case["backward"]:
        outs, grads = [got.log_probs, got.entropy], [_array(s.g_log), _array(s.g_ent)]
        if k:
            outs.append(got.top_log_probs)
            grads.append(_array(s.g_top))
        tg.autograd.backward(outs, grads)
        out["grad"] = _torch(tg.Tensor._wrap(arrived[0]))
    return out


def own_decode(s):
    import tensorgrad_b200 as tg

    return {"out": _torch(tg.paged_attention(_tensor(s.q), _tensor(s.keys), _tensor(s.values), _tensor(s.pages), _tensor(s.lengths)))}


def own_copy(s):
    import tensorgrad_b200 as tg

    tg.copy_pages(_tensor(s.keys), _tensor(s.values), s.src, s.dst)
    return {"keys": s.keys, "values": s.values}


def own_append(s):
    import tensorgrad_b200 as tg

    tg.append_pages(_tensor(s.k), _tensor(s.v), _tensor(s.keys), _tensor(s.values), _tensor(s.pages), _tensor(s.lengths))
    return {"keys": s.keys, "values": s.values}


def own_gather(s):
    import tensorgrad_b200 as tg

    keys, values = tg.gather_pages(_tensor(s.keys), _tensor(s.values), _tensor(s.pages), _tensor(s.lengths), s.longest)
    return {"keys": _torch(keys), "values": _torch(values)}


def own_int8(s):
    import tensorgrad_b200 as tg

    weight = tg.Int8Weight(_array(s.weight), _array(s.scale), s.x.shape[1])
    return {"out": _torch(tg.int8_linear(_tensor(s.x), weight, None if s.bias is None else _tensor(s.bias)))}


# ---------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return globals()["exact_" + s.op](s)


def exact_score(s):
    k = s.case["top_k"]
    parts = []
    for at in range(0, s.case["rows"], 512):
        rows = slice(at, at + 512)
        x = s.logits[rows].double()
        top = x.max(1, keepdim=True).values
        norm = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
        lp = x - norm
        p = torch.exp(lp)
        surprise = torch.where(p > 0, -lp, torch.zeros_like(lp))
        ent = (p * surprise).sum(1)
        t = s.targets[rows]
        live = t >= 0
        one = torch.arange(len(t), device="cuda")
        lt = torch.where(live, lp[one, t.clamp(min=0)], torch.zeros_like(ent))
        out = {"log_probs": lt, "entropy": ent}
        ids = None
        if k:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices
            ids = order[:, :k]
            out["top_log_probs"] = torch.take_along_dim(lp, ids, 1)
        if s.case["backward"]:
            gl = s.g_log[rows].double() * live
            ge = s.g_ent[rows].double()
            # d log_prob / dx_j = [j = t] - p_j;  d entropy / dx_j = p_j (surprise_j - entropy).
            grad = p * (ge[:, None] * (surprise - ent[:, None])) - p * gl[:, None]
            grad[one, t.clamp(min=0)] += gl
            if k:
                gt = s.g_top[rows, :k].double()
                grad -= p * gt.sum(1)[:, None]
                grad.scatter_add_(1, ids, gt)
            out["grad"] = grad
        parts.append(out)
    whole = {key: torch.cat([part[key] for part in parts]) for key in parts[0]}
    if k:
        whole["top_ids"] = None
    return whole


def exact_decode(s):
    c = s.case
    out = torch.zeros(c["batch"], c["kv_heads"] * c["group"], c["width"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(s.lengths.tolist()):
        used = s.pages[b, :-(-n // c["page"])]
        for h in range(c["kv_heads"] if n else 0):
            k = s.keys[used, h].double().reshape(-1, c["width"])[:n]
            v = s.values[used, h].double().reshape(-1, c["width"])[:n]
            heads = slice(h * c["group"], (h + 1) * c["group"])
            a = torch.softmax(s.q[b, heads].double() @ k.T / math.sqrt(c["width"]), 1)
            out[b, heads] = a @ v
    return {"out": out}


def exact_copy(s):
    out = {}
    for name in ("keys", "values"):
        x = getattr(s, name)
        was = x.clone()
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            x[:, b].copy_(was[:, a])
        out[name] = x
    return out


def exact_append(s):
    size = s.case["page"]
    pages, lengths = s.pages.tolist(), s.lengths.tolist()
    for b in range(s.case["batch"]):
        at, end = lengths[b], lengths[b] + s.case["tokens"]
        while at < end:
            upto = min(end, (at // size + 1) * size)
            new, held = slice(at - lengths[b], upto - lengths[b]), slice(at % size, at % size + upto - at)
            s.keys[pages[b][at // size], :, held] = s.k[b, :, new]
            s.values[pages[b][at // size], :, held] = s.v[b, :, new]
            at = upto
    return {"keys": s.keys, "values": s.values}


def exact_gather(s):
    c = s.case
    shape = (c["batch"], c["kv_heads"], c["longest"], c["width"])
    out = {"keys": torch.zeros(shape, dtype=s.keys.dtype, device="cuda"), "values": torch.zeros(shape, dtype=s.keys.dtype, device="cuda")}
    for b, n in enumerate(s.lengths.tolist()):
        used = s.pages[b, :-(-n // c["page"])]
        for h in range(c["kv_heads"] if n else 0):
            out["keys"][b, h, :n] = s.keys[used, h].reshape(-1, c["width"])[:n]
            out["values"][b, h, :n] = s.values[used, h].reshape(-1, c["width"])[:n]
    return out


def exact_int8(s):
    # The integers follow from the inputs' own type (scale and quotient are rounded there); the
    # products and the scaling are in 64 bits.
    k = s.x.shape[1]
    top = s.x.abs().max(1).values
    unit = (top / 127)[:, None]
    q = torch.zeros_like(s.x)
    live = top > 0
    q[live] = (s.x[live] / unit[live]).round().clamp(-127, 127)
    total = q.double() @ s.weight[:, :k].double().T
    y = total * unit.double() * s.scale.double()[None]
    return {"out": y if s.bias is None else y + s.bias.double()}
