"""What the operators of a network's concrete pass cost, and what they have to compute.

Two operators, in the forms in which a network's own answer, its gradient with respect to the embeddings and its
answer at one position are computed:

    attention        softmax(scale q k^T) v over packed sequences of different lengths, grouped heads, causal or not
    residual norm    x + residual, normalised along the row: root mean square, layer norm, or mean subtraction only;
                     optionally written in 8 bits with a scale for each row

`own` chooses between the framework's calls and the plain form: elementary tensor operations in 32 bits, rounded once
at the end.  `exact` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    def attention(name, op, dtype, seqs, shortest, longest, heads, kv_heads, size, causal):
        return {"name": name, "op": op, "dtype": dtype, "seqs": seqs, "shortest": shortest, "longest": longest, "spread": 1,
                "heads": heads, "kv_heads": kv_heads, "size": size, "causal": causal}

    def norm(name, op, dtype, rows, width, kind):
        return {"name": name, "op": op, "dtype": dtype, "rows": rows, "width": width, "kind": kind}

    return [
        # the 30 positions of one 32-word sentence, a copy of the sentence for each, through a layer of 4 heads of 64:
        # the batch that the search for radii steps through
        attention("sentence batch", "attention", "float32", 30, 32, 32, 4, 4, 64, False),
        # a set of documents of different lengths answered in one pass
        attention("packed prompts", "attention", "bfloat16", 8, 150, 4096, 32, 8, 128, True),
        # one long document
        attention("long prompt", "attention", "bfloat16", 1, 16384, 16384, 32, 8, 128, True),
        # one step of the gradient search on the longest sentences of the attention benchmark (L = 128, 4 heads of 64)
        attention("sentence batch, gradient", "attention_train", "float32", 30, 128, 128, 4, 4, 64, False),
        # head size that is no power of two, ragged, both directions of the text
        attention("odd heads, gradient", "attention_train", "float16", 13, 37, 1021, 12, 12, 80, False),
        attention("packed prompts, gradient", "attention_train", "bfloat16", 5, 300, 4096, 32, 8, 128, True),
        # the next word after documents of up to 8192 words
        attention("one word, long caches", "attention_token", "bfloat16", 64, 100, 8192, 32, 8, 128, True),
        # the last layer of a classifier: only the pooled position asks
        attention("pooled position", "attention_token", "float32", 30, 128, 128, 4, 4, 64, False),
        # rows of the sentence batch
        norm("sentence norm", "norm", "float32", 960, 256, "standard"),
        norm("prompt norm", "norm", "bfloat16", 16384, 4096, "rms"),
        norm("prompt norm, gradient", "norm_train", "bfloat16", 8191, 5120, "rms"),
        norm("prompt norm, 8 bits", "norm_8bit", "bfloat16", 4099, 4096, "rms"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention_train", "attention_train", "attention_token", "norm", "norm_train", "norm_8bit"])
    if op.startswith("norm"):
        dtype = rng.choice(["float32", "bfloat16", "float16"]) if op != "norm_8bit" else rng.choice(["bfloat16", "float16"])
        width = _log_uniform(rng, 64, 8192)
        if rng.random() < 0.7:
            width = max(8, width // 8 * 8)
        rows = _log_uniform(rng, 1, max(2, (1 << 26) // width))
        return {"op": op, "dtype": dtype, "rows": rows, "width": width,
                "kind": "rms" if op == "norm_8bit" else rng.choice(["rms", "rms", "standard", "no_var"])}
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    size = rng.choice([32, 64, 64, 80, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    if op == "attention_token":
        longest = _log_uniform(rng, 1, 8192)
        seqs = _log_uniform(rng, 1, 64)
    else:
        longest = _log_uniform(rng, 1, 4096)
        seqs = _log_uniform(rng, 1, max(2, min(64, (1 << 30) // (longest * longest * max(4, heads)))))
    return {"op": op, "dtype": dtype, "seqs": seqs, "shortest": rng.randint(1, longest), "longest": longest,
            "spread": rng.randint(2, 1 << 20), "heads": heads, "kv_heads": kv_heads, "size": size, "causal": rng.random() < 0.5}


def _lengths(case):
    """The sequences' lengths: the longest, and the others anywhere between the shortest and the longest."""
    r = random.Random(case["spread"])
    return [case["longest"]] + [r.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"] - 1)]


def _query_lengths(case):
    return [1] * case["seqs"] if case["op"] == "attention_token" else _lengths(case)


def _pairs(case):
    """How many (query, key) pairs are not masked; the last query stands at the last key."""
    n = 0
    for a, b in zip(_query_lengths(case), _lengths(case)):
        n += sum(max(0, b - a + 1 + i) for i in range(a)) if case["causal"] else a * b
    return n


def work(case):
    if case["op"].startswith("norm"):
        rows, width, es = case["rows"], case["width"], 2 if case["dtype"] != "float32" else 4
        n = rows * width
        if case["op"] == "norm":       # reads x and the residual, writes the sum and the normalised sum
            return {"bytes": 4 * n * es, "flops": 6 * n}
        if case["op"] == "norm_8bit":  # the same with one byte for each normalised value
            return {"bytes": 3 * n * es + n + 4 * rows, "flops": 8 * n}
        # the two gradients that come in and the one that goes out besides
        return {"bytes": 7 * n * es, "flops": 16 * n}
    es = 2 if case["dtype"] != "float32" else 4
    q = sum(_query_lengths(case)) * case["heads"] * case["size"]
    kv = sum(_lengths(case)) * case["kv_heads"] * case["size"]
    product = 2 * _pairs(case) * case["heads"] * case["size"]
    if case["op"] == "attention_train":
        return {"bytes": es * (4 * q + 4 * kv), "flops": 7 * product}
    return {"bytes": es * (2 * q + 2 * kv), "flops": 2 * product}


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    if case["op"].startswith("norm"):
        rows, width = case["rows"], case["width"]
        s = {"x": randn(rows, width), "residual": randn(rows, width),
             "weight": (1 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype),
             "bias": None if case["kind"] == "rms" else (0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype)}
        if case["op"] == "norm_train":
            s.update(dy=randn(rows, width), dsum=randn(rows, width))
        return s
    tq, tk = sum(_query_lengths(case)), sum(_lengths(case))
    s = {"q": randn(tq, case["heads"], case["size"]), "k": randn(tk, case["kv_heads"], case["size"]),
         "v": randn(tk, case["kv_heads"], case["size"])}
    if case["op"] == "attention_train":
        s["dout"] = randn(tq, case["heads"], case["size"])
    return s


def _plain_packing(lengths, key_lengths):
    """Where the rows of a padded batch stand in the packed rows and the other way round."""
    def side(n):
        n = torch.tensor(n, device="cuda")
        starts = torch.cumsum(n, 0) - n
        at = torch.arange(int(n.max()), device="cuda")
        seq = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n)
        inside = at < n[:, None]
        return {"rows": torch.where(inside, starts[:, None] + at, 0), "inside": inside, "seq": seq,
                "pos": torch.arange(len(seq), device="cuda") - starts[seq], "n": n}
    return {"q": side(lengths), "k": side(key_lengths)}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if not case["op"].startswith("norm"):
        if own:
            from faith_amd import ops
            s["packing"] = ops.Packing(_query_lengths(case), _lengths(case), device="cuda")
        else:
            s["packing"] = _plain_packing(_query_lengths(case), _lengths(case))
    return s


# ------------------------------------------------------------------------------------------ the plain forms
def _padded(x, side):
    """Packed [T, heads, size] -> [sequences, heads, length, size] in 32 bits, zero behind each sequence."""
    x = x.float()[side["rows"]]
    return torch.where(side["inside"][:, :, None, None], x, 0.0).transpose(1, 2).contiguous()


def _packed(x, side, dtype):
    return x[side["seq"], :, side["pos"]].to(dtype)


def _plain_probabilities(q, k, packing, causal):
    n, heads, lq, size = q.shape
    kv_heads, lk = k.shape[1], k.shape[2]
    scores = (q * (1.0 / math.sqrt(size))).reshape(n, kv_heads, -1, size) @ k.transpose(2, 3)
    scores = scores.reshape(n, heads, lq, lk)
    masked = ~packing["k"]["inside"][:, None, :]
    if causal:
        # the last query of a sequence stands at its last key
        last = torch.arange(lq, device="cuda")[None, :] + (packing["k"]["n"] - packing["q"]["n"])[:, None]
        masked = masked | (torch.arange(lk, device="cuda") > last[:, :, None])
    scores.masked_fill_(masked[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total == 0, 1.0, total))


def _plain_attention(s):
    case, packing, dtype = s["case"], s["packing"], s["q"].dtype
    q, k, v = _padded(s["q"], packing["q"]), _padded(s["k"], packing["k"]), _padded(s["v"], packing["k"])
    n, heads, lq, size = q.shape
    kv_heads, lk = k.shape[1], k.shape[2]
    p = _plain_probabilities(q, k, packing, case["causal"]).reshape(n, kv_heads, -1, lk)
    out = _packed((p @ v).reshape(n, heads, lq, size), packing["q"], dtype)
    if case["op"] != "attention_train":
        return out
    dout = _padded(s["dout"], packing["q"]).reshape(n, kv_heads, -1, size)
    dv = p.transpose(2, 3) @ dout
    dp = dout @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * (1.0 / math.sqrt(size))
    dq = (ds @ k).reshape(n, heads, lq, size)
    dk = ds.transpose(2, 3) @ q.reshape(n, kv_heads, -1, size)
    return out, _packed(dq, packing["q"], dtype), _packed(dk, packing["k"], dtype), _packed(dv, packing["k"], dtype)


EPS = 1e-6


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    h = s["x"].float() + s["residual"].float()
    centred = h if case["kind"] == "rms" else h - h.mean(-1, keepdim=True)
    r = 1.0 if case["kind"] == "no_var" else torch.rsqrt(centred.square().mean(-1, keepdim=True) + EPS)
    z = centred * r
    y = z * s["weight"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["op"] == "norm":
        return y.to(dtype), h.to(dtype)
    if case["op"] == "norm_8bit":
        scale = y.abs().amax(-1, keepdim=True) / 448.0
        q = (y / torch.where(scale == 0, 1.0, scale)).to(torch.float8_e4m3fn)
        return (q.float() * scale).to(dtype), h.to(dtype)
    dy = s["dy"].float()
    g = dy * s["weight"].float()
    dh = g
    if case["kind"] != "no_var":
        dh = dh - z * (g * z).mean(-1, keepdim=True)
    if case["kind"] != "rms":
        dh = dh - g.mean(-1, keepdim=True)
    got = [y.to(dtype), h.to(dtype), (s["dsum"].float() + dh * r).to(dtype), (dy * z).sum(0).to(dtype)]
    if s["bias"] is not None:
        got.append(dy.sum(0).to(dtype))
    return got


# ------------------------------------------------------------------------------------------ the framework's calls
def _own_attention(s):
    from faith_amd import ops
    case = s["case"]
    if case["op"] != "attention_train":
        return ops.attention(s["q"], s["k"], s["v"], s["packing"], causal=case["causal"])
    out, lse = ops.attention(s["q"], s["k"], s["v"], s["packing"], causal=case["causal"], return_lse=True)
    return (out, *ops.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["packing"], causal=case["causal"]))


def _own_norm(s):
    from faith_amd import ops
    case = s["case"]
    if case["op"] == "norm":
        return ops.residual_norm(s["x"], s["residual"], s["weight"], s["bias"], case["kind"], EPS)
    if case["op"] == "norm_8bit":
        q, scale, h = ops.residual_norm(s["x"], s["residual"], s["weight"], s["bias"], case["kind"], EPS, quantize="e4m3")
        return (q.float() * scale[:, None]).to(h.dtype), h
    y, h, stats = ops.residual_norm(s["x"], s["residual"], s["weight"], s["bias"], case["kind"], EPS, return_stats=True)
    dx, dweight, dbias = ops.residual_norm_backward(s["dy"], h, s["weight"], stats, case["kind"], dsum=s["dsum"],
                                                    with_bias=s["bias"] is not None)
    return [y, h, dx, dweight] + ([dbias] if s["bias"] is not None else [])


def run(state):
    if state["case"]["op"].startswith("norm"):
        return _own_norm(state) if own else _plain_norm(state)
    return _own_attention(state) if own else _plain_attention(state)


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_attention(case, s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    group, size = case["heads"] // case["kv_heads"], case["size"]
    train = case["op"] == "attention_train"
    out = torch.zeros_like(q)
    grads = (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v))
    a = b = 0
    for nq, nk in zip(_query_lengths(case), _lengths(case)):
        i = torch.arange(nq, device="cuda")[:, None] + (nk - nq)
        allowed = torch.arange(nk, device="cuda")[None, :] <= (i if case["causal"] else nk)
        for h in range(case["heads"]):
            qh, kh, vh = q[a:a + nq, h], k[b:b + nk, h // group], v[b:b + nk, h // group]
            logits = torch.mm(qh, kh.t()) / math.sqrt(size)
            logits = torch.where(allowed, logits, -math.inf)
            p = torch.nan_to_num(torch.softmax(logits, dim=1), nan=0.0)
            out[a:a + nq, h] = torch.mm(p, vh)
            if train:
                do = s["dout"][a:a + nq, h].double()
                delta = (do * out[a:a + nq, h]).sum(1, keepdim=True)
                ds = p * (torch.mm(do, vh.t()) - delta) / math.sqrt(size)
                grads[0][a:a + nq, h] = torch.mm(ds, kh)
                grads[1][b:b + nk, h // group] += torch.mm(ds.t(), qh)
                grads[2][b:b + nk, h // group] += torch.mm(p.t(), do)
        a, b = a + nq, b + nk
    return (out, *grads) if train else out


def _exact_norm(case, s):
    x, r, w = s["x"].double(), s["residual"].double(), s["weight"].double()
    b = s["bias"].double() if s["bias"] is not None else None
    h = x + r
    mean = 0.0 if case["kind"] == "rms" else h.sum(1, keepdim=True) / h.shape[1]
    spread = ((h - mean) ** 2).sum(1, keepdim=True) / h.shape[1] + EPS
    inverse = torch.ones_like(spread) if case["kind"] == "no_var" else 1.0 / spread.sqrt()
    unit = (h - mean) * inverse
    y = unit * w if b is None else unit * w + b
    if case["op"] == "norm":
        return y, h
    if case["op"] == "norm_8bit":
        scale = y.abs().max(dim=1, keepdim=True).values / 448.0
        t = y / torch.where(scale == 0, torch.ones_like(scale), scale)
        # the values of one sign bit, four exponent bits and three mantissa bits: steps of 2^(e - 3), not below 2^-9
        e = torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
        step = torch.exp2(e - 3.0)
        return torch.round(t / step) * step * scale, h
    dy, n = s["dy"].double(), h.shape[1]
    dunit = dy * w
    dh = dunit * inverse
    if case["kind"] != "rms":
        dh = dh - dunit.sum(1, keepdim=True) * inverse / n
    if case["kind"] != "no_var":
        dh = dh - (h - mean) * inverse ** 3 * (dunit * (h - mean)).sum(1, keepdim=True) / n
    got = [y, h, s["dsum"].double() + dh, (dy * unit).sum(0)]
    return got if b is None else got + [dy.sum(0)]


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_norm(case, s) if case["op"].startswith("norm") else _exact_attention(case, s)
