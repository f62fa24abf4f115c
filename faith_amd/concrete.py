"""The network itself: its answer, the gradient of its answer, and the radius at which the answer breaks.

`forward.py` propagates bounds through a network; this module runs the same network on numbers.  The dense layers are plain
matrix products, attention and the residual norms are this library's kernels (`ops.attention`, `ops.residual_norm`),
differentiable here.  Sentences of different lengths go through together, packed one behind the other without padding
(`ops.Packing`); attention is the only place where it shows.

    logits, predict         the network's answer for a batch of sentences; what `forward.verify_safety(..., label=None)` and
                            `forward.certified_radii(..., label=None)` take as the label that has to survive
    adversarial_radii       the smallest radius at which a search by gradients finds a perturbation that changes the answer:
                            the other side of `forward.certified_radii`

Networks are the objects that `forward.py` describes (`.embedding_norm`, `.layers`, `.pooler`, `.classifier`, `.layer_norm`,
`.hidden_act`), with three additions that bounds are not propagated through: `.layer_norm = "rms"`, `.causal = True`, and
layers whose `attention.self.num_key_value_heads` is smaller than `num_attention_heads`.  Embeddings and parameters are
float32, bfloat16 or float16 alike.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import ops

# what Bounds.layer_norm adds to the variance in mode "standard"
EPS = {"standard": 1e-12, "rms": 1e-6, "no_var": 0.0}


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packing, causal, scale):
        out, lse = ops.attention(q, k, v, packing, causal, scale, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.rest = (packing, causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        return (*ops.attention_backward(dout.contiguous(), q, k, v, out, lse, *ctx.rest), None, None, None)


def attention(q, k, v, packing, causal=False, scale=None):
    """ops.attention, differentiable with respect to q, k and v (not the scale, which is a number), for heads of any size up to 128
    (one that does not fall into whole groups of 16 bytes is carried with zeros behind it)."""
    if isinstance(scale, torch.Tensor):
        if torch.is_grad_enabled() and scale.requires_grad:
            raise ValueError("scale: has no gradient here; multiply q by it")
        scale = float(scale)                              # the gradient's scale is that of this call, whatever the tensor holds by then
    causal = bool(causal)
    size, per = q.shape[2], 16 // q.element_size()
    if size % per and size < 128:
        if scale is None:
            scale = 1.0 / math.sqrt(size)
        q, k, v = (torch.nn.functional.pad(t, (0, per - size % per)) for t in (q, k, v))
        return attention(q, k, v, packing, causal, scale)[:, :, :size]
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, packing, causal, scale)
    return ops.attention(q, k, v, packing, causal, scale)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, kind, eps):
        y, h, stats = ops.residual_norm(x, residual, weight, bias, kind, eps, return_stats=True)
        ctx.save_for_backward(h, weight, stats)
        ctx.kind = kind
        ctx.set_materialize_grads(False)
        # without a residual the sum is x: a view of it would be an output that is an input
        return y, h if residual is not None else h.detach()

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum):
        h, weight, stats = ctx.saved_tensors
        _, with_residual, with_weight, with_bias = ctx.needs_input_grad[:4]
        if dy is None:
            return dsum, dsum if with_residual else None, None, None, None, None
        dx, dweight, dbias = ops.residual_norm_backward(dy.contiguous(), h, weight, stats, ctx.kind, None if dsum is None else dsum.contiguous(),
                                                        with_weight, with_bias)
        return dx, dx if with_residual else None, dweight, dbias, None, None


def residual_norm(x, residual=None, weight=None, bias=None, kind="rms", eps=1e-6):
    """ops.residual_norm without its 8-bit form, differentiable with respect to all four tensors; returns (y, h)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        return _ResidualNorm.apply(x, residual, weight, bias, kind, eps)
    return ops.residual_norm(x, residual, weight, bias, kind, eps)


def _norm(x, residual, normalizer, layer_norm, activations):
    if layer_norm == "no":
        return x if residual is None else x + residual
    weight, bias = normalizer.weight, getattr(normalizer, "bias", None)
    if activations is None:
        return residual_norm(x, residual, weight, bias, layer_norm, EPS[layer_norm])[0]
    q, scales, _ = ops.residual_norm(x, residual, weight, bias, layer_norm, EPS[layer_norm], quantize=activations)
    return (q.float() * scales[:, None]).to(x.dtype)


def _dense(x, layer):
    return torch.nn.functional.linear(x, layer.weight, layer.bias)


def _act(x, name):
    if name == "relu":
        return torch.relu(x)
    if name == "tanh":
        return torch.tanh(x)
    raise NotImplementedError(name)


def encoder_layer(x, layer, packing, layer_norm="no_var", hidden_act="relu", causal=False, activations=None, queries=None):
    """One layer on packed rows x [tokens, hidden]: attention block, residual + norm, feed-forward, residual + norm
    (forward.bound_layer on numbers).  queries: (rows of x, a Packing of them against x's keys) when only some positions
    ask -- the last layer in front of a pooler."""
    att = layer.attention.self
    heads, size = att.num_attention_heads, att.attention_head_size
    kv_heads = getattr(att, "num_key_value_heads", None) or heads
    asking = x if queries is None else x[queries[0]]
    q = _dense(asking, att.query).view(-1, heads, size)
    k, v = _dense(x, att.key).view(-1, kv_heads, size), _dense(x, att.value).view(-1, kv_heads, size)
    context = attention(q, k, v, packing if queries is None else queries[1], causal).reshape(-1, heads * size)
    x = _norm(_dense(context, layer.attention.output.dense), asking, layer.attention.output.LayerNorm, layer_norm, activations)
    y = _dense(_act(_dense(x, layer.intermediate.dense), hidden_act), layer.output.dense)
    return _norm(y, x, layer.output.LayerNorm, layer_norm, activations)


class Batch:
    """The lengths of a batch of sentences as `logits` and `predict` take them, kept by a caller who asks more than once:
    the packing of all positions, and that of the first of each against all."""

    def __init__(self, lengths, device):
        self.packing = ops.Packing(lengths, device=device)
        if min(self.packing.lengths) == 0:
            raise ValueError("a sentence without words has no first position to pool")
        self.first = torch.tensor(self.packing.starts()[:-1], dtype=torch.int64, device=device)
        self.pooled = ops.Packing([1] * len(self.packing.lengths), self.packing.lengths, device=device)


def _rows_of(embeddings, lengths):
    """([tokens, hidden], Batch) from one tensor [sentences, L, hidden], or from packed rows and their lengths."""
    if embeddings.dim() == 3 and lengths is None:
        return embeddings.reshape(-1, embeddings.shape[2]), Batch([embeddings.shape[1]] * embeddings.shape[0], embeddings.device)
    if embeddings.dim() == 2 and lengths is not None:
        batch = lengths if isinstance(lengths, Batch) else Batch(lengths, embeddings.device)
        if batch.packing.tokens != embeddings.shape[0]:
            raise ValueError(f"{embeddings.shape[0]} rows, {batch.packing.tokens} words")
        return embeddings, batch
    raise ValueError("embeddings: [sentences, length, hidden], or packed [words, hidden] with the sentences' lengths")


def _logits(network, x, batch, activations=None):
    causal = bool(getattr(network, "causal", False))
    if network.embedding_norm is not None:
        x = _norm(x, None, network.embedding_norm, network.layer_norm, activations)
    for i, layer in enumerate(network.layers):
        # only the first position of each sentence goes on to the pooler: in the last layer nothing else asks.  (A causal
        # network's first position sees itself alone, which is the whole layer's business.)
        last = i == len(network.layers) - 1 and not causal
        x = encoder_layer(x, layer, batch.packing, network.layer_norm, network.hidden_act, causal, activations,
                          (batch.first, batch.pooled) if last else None)
    if causal or not network.layers:
        x = x[batch.first]
    return _dense(torch.tanh(_dense(x, network.pooler)), network.classifier)


def logits(network, embeddings, lengths=None, activations=None):
    """The network's output [sentences, classes] for embeddings [sentences, L, hidden], or packed [words, hidden] with the
    sentences' lengths (a list, or a Batch that the caller keeps).  Differentiable.  activations "int8" / "e4m3": what leaves a normalisation is held in 8 bits
    with a scale for each row, as a network deployed that way would hold it (no gradient)."""
    if activations is not None and activations not in ops._BITS:
        raise ValueError(f"activations={activations!r}: one of {', '.join(ops._BITS)} or None")
    rows, batch = _rows_of(embeddings, lengths)
    if activations is not None:
        with torch.no_grad():
            return _logits(network, rows.contiguous(), batch, activations)
    return _logits(network, rows.contiguous(), batch)


def predict(network, embeddings, lengths=None, activations=None):
    """The class that the network answers for each sentence: a list of ints."""
    with torch.no_grad():
        return logits(network, embeddings, lengths, activations).argmax(-1).tolist()


def _steepest(g, p):
    """The direction of unit p-norm along which the linear function g grows most, per row of g [n, dim]."""
    if math.isinf(p) or p >= 10:                          # p >= 10 is infinity, as in the propagation
        return torch.sign(g)
    if p == 1:
        best = g.abs().argmax(1, keepdim=True)
        return torch.zeros_like(g).scatter_(1, best, torch.sign(g.gather(1, best)))
    q = p / (p - 1)
    d = torch.sign(g) * (g.abs() / g.abs().amax(1, keepdim=True).clamp_min(1e-30)).pow(q - 1)
    return d / torch.linalg.vector_norm(d, ord=p, dim=1, keepdim=True).clamp_min(1e-30)


def _into_ball(d, p, radii):
    if math.isinf(p) or p >= 10:
        return torch.maximum(torch.minimum(d, radii[:, None]), -radii[:, None])
    # a little further in than the norm's own rounding may be off
    inside = radii * (1 - 2.0 ** -40) if d.dtype == torch.float64 else radii
    return d * (inside / torch.linalg.vector_norm(d, ord=p, dim=1).clamp_min(1e-30)).clamp_max(1.0)[:, None]


def _toward(t, base):
    """For every element of t the neighbour of its type that lies one step closer to `base`."""
    kind = torch.int32 if t.element_size() == 4 else torch.int16
    bits = t.view(kind)                                   # sign and magnitude: one less is one step towards zero
    step = torch.where((t > 0) == (base < t), bits - 1, bits + 1)
    smallest = torch.where(base < 0, torch.iinfo(kind).min + 1, 1)
    return torch.where(t == 0, smallest, step).to(kind).view(t.dtype)


def _moved(base, delta):
    """base + delta (float64) in base's type, rounded to nearest but never past delta: every element moves by delta's at most, so the
    perturbation that the network sees has no norm larger than delta's."""
    moved = (base.double() + delta).to(base.dtype)
    past = (moved.double() - base.double()).abs() > delta.abs()
    return torch.where(past, _toward(moved, base), moved)


def falsify(network, embeddings, positions, radii, label, p=2.0, steps=10, batch=None):
    """Searches, for every (position, radius) pair at once, for a perturbation of the embedding at that position, of p-norm at
    most the radius, with which the network no longer answers `label` with a positive margin: `steps` steps of projected steepest ascent from the
    sentence itself.  embeddings [1, L, hidden].  Returns a list of bools; True is a proof, False only that none was found: what counts is
    the perturbation of the embeddings as they are, rounded to their type (in 16 bits a radius under half a step of every element holds none
    but zero), and a margin that is a finite number.

    A step is one pass forward and backward over as many copies of the sentence as there are pairs.  batch: their Batch,
    where the caller keeps one."""
    from .forward import _checked_positions
    if len(radii) != len(positions):
        raise ValueError(f"{len(positions)} positions, {len(radii)} radii")
    if not p >= 1:
        raise ValueError(f"p={p}: the perturbation norm must be >= 1")
    if steps < 0:
        raise ValueError(f"{steps} steps")
    for r in radii:
        if not 0 <= r < math.inf:
            raise ValueError(f"radius {r!r} is not a radius")
    if not positions:
        return []
    if embeddings.dim() != 3 or embeddings.shape[0] != 1:
        raise ValueError(f"embeddings: expected one sentence [1, length, hidden], got {tuple(embeddings.shape)}")
    n, length = len(positions), embeddings.shape[1]
    at = [g[0] for g in _checked_positions([[i] for i in positions], length)]
    classes = network.classifier.weight.shape[0]
    if label != int(label) or not 0 <= label < classes:
        raise ValueError(f"label {label!r}: the network answers with one of {classes} classes")
    label = int(label)
    dev = embeddings.device
    batch = batch or Batch([length] * n, dev)
    if batch.packing.lengths != (length,) * n:
        raise ValueError(f"batch: expected {n} sentences of {length}")
    base = embeddings.detach().expand(n, length, embeddings.shape[2]).reshape(n * length, -1)
    where = batch.first + torch.tensor(at, dtype=torch.int64, device=dev)
    r = torch.tensor([float(v) for v in radii], dtype=torch.float64, device=dev)
    delta = torch.zeros(n, base.shape[1], dtype=torch.float64, device=dev)
    found = torch.zeros(n, dtype=torch.bool, device=dev)
    for step in range(steps + 1):
        with torch.enable_grad():
            # leaf: the perturbed rows, so that the parameters collect no gradients
            moved = _moved(base[where], delta).requires_grad_(True)
            out = _logits(network, base.index_copy(0, where, moved), batch).float()
            others = out.index_fill(1, torch.tensor([label], device=dev), -math.inf).amax(1)
            margin = out[:, label] - others
            # as in the propagation: an answer is safe only while its margin is positive.  NaN or an infinity is no answer: an
            # overflow of the arithmetic, which proves nothing
            found |= (margin.detach() <= 0) & torch.isfinite(margin.detach())
            if step == steps:
                break
            (g,) = torch.autograd.grad(margin.sum(), moved)
        # a first step to the border, then ones that can cross the ball; none along a gradient that is no number
        size = r if step == 0 else r * (2.0 / steps)
        usable = torch.isfinite(g).all(1, keepdim=True)
        delta = torch.where(usable, _into_ball(delta - _steepest(g.float(), p).double() * size[:, None], p, r), delta)
    return found.tolist()


def adversarial_radii(network, embeddings, positions, label=None, p=2.0, max_eps=0.1, num_iters=10, steps=10):
    """For every position the smallest radius at which `falsify` succeeds: max_eps and then num_iters bisections below it, as
    in forward.certified_radii; infinity where max_eps does not break the answer.  No radius under the certified one comes
    out, and the truth lies between the two.  label: default the network's own answer."""
    if label is None:
        (label,) = predict(network, embeddings)
    n = len(positions)
    batch = Batch([embeddings.shape[1]] * n, embeddings.device) if n else None
    broken = falsify(network, embeddings, positions, [float(max_eps)] * n, label, p, steps, batch)
    lo, hi = [0.0] * n, [float(max_eps) if b else math.inf for b in broken]
    for _ in range(num_iters if any(broken) else 0):
        # positions that held at max_eps are only carried along: all of them share every launch
        mid = [float(max_eps) if math.isinf(h) else (l + h) / 2 for l, h in zip(lo, hi)]
        for i, b in enumerate(falsify(network, embeddings, positions, mid, label, p, steps, batch)):
            if math.isinf(hi[i]):
                continue
            if b:
                hi[i] = mid[i]
            else:
                lo[i] = mid[i]
    return hi
