"""The concrete pass as it is used: a network's answers, their gradient, and the radii on both sides of the truth."""
import math
from types import SimpleNamespace

import pytest
import torch

from faith_amd.workloads import random_layer, to_device
from tests.oracle_bounds import true_layer

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, INTER = 64, 4, 128


def network(seed, mode, layers=2, hidden=HIDDEN, heads=HEADS, inter=INTER, classes=2, device="cuda", **more):
    g = torch.Generator().manual_seed(seed)
    lin = lambda o, i: SimpleNamespace(weight=torch.randn(o, i, generator=g) / i ** 0.5, bias=0.05 * torch.randn(o, generator=g))
    norm = SimpleNamespace(weight=1 + 0.1 * torch.randn(hidden, generator=g), bias=0.05 * torch.randn(hidden, generator=g))
    net = SimpleNamespace(embedding_norm=norm, layers=[random_layer(g, hidden, heads, inter) for _ in range(layers)], pooler=lin(hidden, hidden),
                          classifier=lin(classes, hidden), layer_norm=mode, hidden_act="relu", **more)
    net.layers = [to_device(l, device) for l in net.layers]
    for k in ("embedding_norm", "pooler", "classifier"):
        setattr(net, k, to_device(getattr(net, k), device))
    return net


def plain_logits(net, x):
    """One sentence [L, hidden] in float64, differentiable."""
    mode, causal = net.layer_norm, getattr(net, "causal", False)

    def ln(v, n):
        if mode == "no":
            return v
        c = v if mode == "rms" else v - v.mean(-1, keepdim=True)
        if mode != "no_var":
            c = c / torch.sqrt((c * c).mean(-1, keepdim=True) + (1e-6 if mode == "rms" else 1e-12))
        return c * n.weight.double() + n.bias.double()
    lin = lambda v, l: v @ l.weight.double().t() + l.bias.double()
    h = ln(x, net.embedding_norm)
    for layer in net.layers:
        a = layer.attention.self
        heads, size = a.num_attention_heads, a.attention_head_size
        kv = getattr(a, "num_key_value_heads", heads)
        L = h.shape[0]
        q = lin(h, a.query).view(L, heads, size).transpose(0, 1)
        k, v = (lin(h, p).view(L, kv, size).transpose(0, 1).repeat_interleave(heads // kv, 0) for p in (a.key, a.value))
        s = q @ k.transpose(1, 2) / math.sqrt(size)
        if causal:
            s = s.masked_fill(torch.ones(L, L, device=x.device).triu(1).bool(), -math.inf)
        c = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(L, -1)
        att = ln(lin(c, layer.attention.output.dense) + h, layer.attention.output.LayerNorm)
        h = ln(lin(torch.relu(lin(att, layer.intermediate.dense)), layer.output.dense) + att, layer.output.LayerNorm)
    return lin(torch.tanh(lin(h[0], net.pooler)), net.classifier)


def sentences(lengths, seed, hidden=HIDDEN):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, hidden, generator=g).cuda() for n in lengths]


# Some 25 operators behind each other, each a few roundings of 32 bits (6e-8) off, times a condition of some ten: 1e-4 leaves
# a factor over that and is far under what a wrong operator makes (order one).
@pytest.mark.parametrize("mode", ["no_var", "standard", "rms", "no"])
@pytest.mark.parametrize("more", [{}, dict(causal=True), dict(kv_heads=2), dict(kv_heads=1, causal=True)])
def test_logits_of_packed_sentences(mode, more):
    from faith_amd import concrete
    more = dict(more)
    kv = more.pop("kv_heads", HEADS)
    net = network(3, mode, **more)
    for layer in net.layers:
        a = layer.attention.self
        a.num_key_value_heads = kv
        for p in (a.key, a.value):
            p.weight, p.bias = p.weight[:kv * HIDDEN // HEADS].contiguous(), p.bias[:kv * HIDDEN // HEADS].contiguous()
    if mode == "no":
        for layer in net.layers:                      # nothing keeps the size of the rows in check
            layer.output.dense.weight *= 0.3
    lengths = [5, 32, 1, 70]
    xs = sentences(lengths, 4)
    got = concrete.logits(net, torch.cat(xs), lengths)
    want = torch.stack([plain_logits(net, x.double()) for x in xs])
    assert got.shape == (4, 2) and float((got.double() - want).abs().max()) <= 1e-4 * max(1.0, float(want.abs().max()))
    batch = concrete.Batch(lengths, "cuda")
    assert torch.equal(concrete.logits(net, torch.cat(xs), batch), got)
    assert concrete.predict(net, torch.cat(xs), batch) == want.argmax(1).tolist()
    one = concrete.logits(net, xs[1][None])
    assert float((one - got[1]).abs().max()) <= 1e-4 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("size", [16, 18])
def test_one_layer_is_the_network_of_the_bounds(size):
    """The network that the soundness tests of the propagation compare with (tests/oracle_bounds.py); heads of 18 are carried
    in whole 16-byte groups."""
    from faith_amd import concrete
    for mode in ("no_var", "standard"):
        net = network(5, mode, layers=1, hidden=4 * size)
        x = sentences([9], 6, 4 * size)[0]
        cpu = to_device(SimpleNamespace(**vars(net)), "cpu")
        layer = to_device(net.layers[0], "cpu")
        _, margin = true_layer(x.cpu().double()[None], layer, cpu.embedding_norm, mode, cpu.pooler, cpu.classifier)
        got = concrete.logits(net, x[None])[0]
        assert abs(float(got[0] - got[1]) - float(margin[0, 0])) <= 1e-4


@pytest.mark.parametrize("mode", ["no_var", "standard", "rms"])
@pytest.mark.parametrize("causal", [False, True])
def test_gradient_of_the_embeddings_and_of_the_parameters(mode, causal):
    from faith_amd import concrete
    net = network(7, mode, causal=causal)
    lengths = [6, 40, 3]
    xs = sentences(lengths, 8)
    params = [net.layers[0].attention.self.value.weight, net.layers[1].attention.output.LayerNorm.weight, net.layers[0].output.LayerNorm.bias,
              net.embedding_norm.weight]
    for t in params:
        t.requires_grad_(True)
    rows = torch.cat(xs).requires_grad_(True)
    w = torch.tensor([[1.0, -0.5], [0.3, 2.0], [-1.0, 0.7]], device="cuda")
    got = torch.autograd.grad((concrete.logits(net, rows, lengths) * w).sum(), [rows] + params)
    rows64 = torch.cat(xs).double().requires_grad_(True)
    out, at = 0.0, 0
    for i, n in enumerate(lengths):
        out = out + (plain_logits(net, rows64[at:at + n]) * w[i].double()).sum()
        at += n
    want = torch.autograd.grad(out, [rows64] + params)
    for a, b in zip(got, want):
        assert float((a.double() - b.double()).norm()) <= 1e-4 * float(b.double().norm())


def test_half_precision_and_eight_bit_activations():
    from faith_amd import concrete
    net = network(9, "standard", hidden=128)
    lengths = [30, 64]
    xs = sentences(lengths, 10, 128)
    want = torch.stack([plain_logits(net, x.double()) for x in xs])
    scale = max(1.0, float(want.abs().max()))
    low = SimpleNamespace(**vars(net))
    cast = lambda o, t: SimpleNamespace(**{k: cast(v, t) for k, v in vars(o).items()}) if isinstance(o, SimpleNamespace) else (o.to(t) if isinstance(o, torch.Tensor) else o)
    # two layers of roundings of 2^-9 (bf16), 2^-12 (fp16), 2^-4 of a value (e4m3) and 1 / 254 of a row's largest (int8)
    for dtype, tol in ((torch.bfloat16, 0.1), (torch.float16, 0.0125)):
        low.embedding_norm, low.pooler, low.classifier = (cast(getattr(net, k), dtype) for k in ("embedding_norm", "pooler", "classifier"))
        low.layers = [cast(l, dtype) for l in net.layers]
        got = concrete.logits(low, torch.cat(xs).to(dtype), lengths)
        assert got.dtype == dtype and float((got.double() - want).abs().max()) <= tol * scale
    for bits, tol in (("int8", 0.1), ("e4m3", 0.5)):
        got = concrete.logits(net, torch.cat(xs), lengths, activations=bits)
        off = float((got.double() - want).abs().max())
        assert 0 < off <= tol * scale


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_the_truth_lies_between_the_radii(p):
    from faith_amd import BoundsMaker, concrete
    from faith_amd import forward as F
    net = network(11, "no_var", layers=1, hidden=32)
    emb = sentences([6], 12, 32)[0][None]
    make = BoundsMaker(SimpleNamespace(perturbed_words=1))
    (label,) = concrete.predict(net, emb)
    positions = [1, 2, 3, 4]
    most = {1.0: 20.0, 2.0: 8.0, math.inf: 3.0}[p]
    low = F.certified_radii(make, net, emb, positions, None, p, most, 8, batched=True)
    assert low == F.certified_radii(make, net, emb, positions, label, p, most, 8, batched=True)
    high = concrete.adversarial_radii(net, emb, positions, None, p, most, 8)
    assert all(0 <= a <= b for a, b in zip(low, high))
    assert any(math.isfinite(h) for h in high)
    for pos, h in zip(positions, high):
        if math.isfinite(h):
            assert concrete.falsify(net, emb, [pos], [h], label, p) == [True]
            assert not F.verify_safety(make, net, emb, pos, h, None, p)
    # nothing breaks inside a certified radius
    assert not any(concrete.falsify(net, emb, positions, [0.999 * a for a in low], label, p))
    assert F.verify_safety_batch(make, net, emb, positions, [0.5 * a for a in low], None, p) == F.verify_safety_batch(make, net, emb, positions, [0.5 * a for a in low], label, p)


def test_label_of_the_network_in_a_captured_propagation():
    from faith_amd import BoundsMaker, concrete
    from faith_amd import forward as F
    net = network(13, "no_var", layers=1, hidden=32)
    emb = sentences([6], 14, 32)[0][None]
    make = BoundsMaker(SimpleNamespace(perturbed_words=1))
    (label,) = concrete.predict(net, emb)
    own, given = F.CapturedVerifier(make, net, emb, 2, None), F.CapturedVerifier(make, net, emb, 2, label)
    for r in (0.001, 0.05, 2.0):
        assert own([1, 3], [r, r]) == given([1, 3], [r, r])


def test_parameters_collect_no_gradients_in_the_search():
    from faith_amd import concrete
    net = network(15, "standard", layers=1)
    for t in (net.classifier.weight, net.layers[0].attention.self.query.weight, net.layers[0].output.LayerNorm.weight):
        t.requires_grad_(True)
    emb = sentences([8], 16)[0][None]
    concrete.adversarial_radii(net, emb, [1, 2], None, 2.0, 4.0, 2, 3)
    assert net.classifier.weight.grad is None and net.layers[0].output.LayerNorm.weight.grad is None
    with torch.no_grad():
        assert len(concrete.falsify(net, emb, [1], [1.0], 0)) == 1


def test_second_derivatives_are_refused():
    from faith_amd import concrete, ops
    x = torch.randn(6, 2, 16, device="cuda", requires_grad=True)
    out = concrete.attention(x, x, x, ops.Packing([6]))
    (g,) = torch.autograd.grad(out.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    y, _ = concrete.residual_norm(x.view(6, 32), None, None, None, "rms")
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_sum_and_normalised_sum_both_carry_gradients():
    """What a network with the norm in front of its blocks does: the sum goes on beside its normalisation."""
    from faith_amd import concrete
    g = torch.Generator(device="cuda").manual_seed(3)
    t = [torch.randn(9, 64, generator=g, device="cuda", requires_grad=True) for _ in range(2)] + [torch.randn(64, generator=g, device="cuda", requires_grad=True) for _ in range(2)]
    for kind in ("rms", "standard", "no_var"):
        for given in ([0, 1, 2, 3], [0, 2, 3], [0]):
            args = [t[i] if i in given else None for i in range(4)]
            y, h = concrete.residual_norm(*args, kind, 1e-6)
            got = torch.autograd.grad((y * y).sum() + (h * h * h).sum(), [t[i] for i in given])
            a = [x.detach().double().requires_grad_(True) if x is not None else None for x in args]
            s = a[0] if a[1] is None else a[0] + a[1]
            c = s if kind == "rms" else s - s.mean(-1, keepdim=True)
            z = c if kind == "no_var" else c / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            yy = z if a[2] is None else z * a[2] + a[3]
            want = torch.autograd.grad((yy * yy).sum() + (s * s * s).sum(), [a[i] for i in given])
            assert all(float((p.double() - q).norm()) <= 1e-5 * float(q.norm()) for p, q in zip(got, want)), (kind, given)
            only = torch.autograd.grad(concrete.residual_norm(*args, kind, 1e-6)[1].square().sum(), t[0])[0]
            assert float((only.double() - 2 * s.detach()).norm()) <= 1e-5 * float(s.detach().norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("p", [2.0, math.inf])
def test_what_breaks_the_answer_in_half_precision_lies_in_the_ball(monkeypatch, dtype, p):
    """Radii near one step of the type: every row that the network is asked about is within its radius of the sentence."""
    from faith_amd import concrete
    net = network(21, "no_var", layers=1, hidden=64)
    cast = lambda o: SimpleNamespace(**{k: cast(v) for k, v in vars(o).items()}) if isinstance(o, SimpleNamespace) else (o.to(dtype) if isinstance(o, torch.Tensor) else o)
    net.embedding_norm, net.pooler, net.classifier, net.layers = cast(net.embedding_norm), cast(net.pooler), cast(net.classifier), [cast(l) for l in net.layers]
    emb = sentences([6], 22, 64)[0][None].to(dtype)
    (label,) = concrete.predict(net, emb)
    radii, seen, run = [0.0, 1e-3, 0.01, 0.05, 1.0, 100.0], [], concrete._logits

    def watched(network, x, batch, activations=None):
        seen.append(x.detach().view(len(radii), 6, 64)[:, 2].double() - emb[0, 2].double())
        return run(network, x, batch, activations)
    monkeypatch.setattr(concrete, "_logits", watched)
    found = concrete.falsify(net, emb, [2] * len(radii), radii, label, p)
    assert not found[0] and len(seen) == 11
    for d in seen:
        assert bool((torch.linalg.vector_norm(d, ord=p, dim=1) <= torch.tensor(radii, device="cuda", dtype=torch.float64)).all())


def test_eight_bit_activations_do_not_hide_what_is_no_number():
    from faith_amd import concrete
    net = network(9, "standard", hidden=128)
    xs = sentences([30, 64], 10, 128)
    xs[0][4, 7] = math.nan
    for bits in (None, "int8", "e4m3"):
        got = concrete.logits(net, torch.cat(xs), [30, 64], activations=bits)
        assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())


def test_none_for_shared_key_heads_is_no_sharing():
    from faith_amd import concrete
    net = network(3, "no_var")
    x = sentences([9], 4)[0][None]
    want = concrete.logits(net, x)
    for layer in net.layers:
        layer.attention.self.num_key_value_heads = None
    assert torch.equal(concrete.logits(net, x), want)
