"""The concrete pass on the host: work items, refusals, the C ABI's argument checks.  No GPU is needed."""
import ctypes
import math
import random

import pytest
import torch

from faith_amd import _lib, concrete, forward, ops


def plan(lengths, key_lengths, heads, kv_heads, element_size, causal, which, size=64):
    n = len(lengths)
    ql, kl, counts = (ctypes.c_int * n)(*lengths), (ctypes.c_int * n)(*key_lengths), (ctypes.c_longlong * 4)()
    args = (ctypes.addressof(ql), ctypes.addressof(kl), n, heads, kv_heads, element_size, size, int(causal), which)
    _lib.call("faith_attention_plan", *args, None, 0, ctypes.addressof(counts))
    total = counts[0] + counts[1]
    out = torch.full((total + 1, 8), -7, dtype=torch.int32)
    _lib.call("faith_attention_plan", *args, out.data_ptr(), total, ctypes.addressof(counts))
    assert bool((out[total] == -7).all())
    rows = out.tolist()
    return rows[:counts[0]], rows[counts[0]:total], counts[2], counts[3]


CASES = [([5], [5], 4, 4), ([1, 1, 1], [700, 3, 65], 8, 2), ([130, 0, 7], [300, 5, 0], 2, 1), ([40, 9], [10, 9], 3, 1),
         ([1], [8192], 32, 8), ([4096] * 9, [4096] * 9, 8, 8), ([1000, 33], [1000, 33], 12, 4), ([128], [16384], 8, 1), ([1] * 70, list(range(70)), 4, 4)]


@pytest.mark.parametrize("lengths, key_lengths, heads, kv_heads", CASES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("element_size", [2, 4])
def test_forward_items_cover_every_row_and_key_once(lengths, key_lengths, heads, kv_heads, causal, element_size):
    items, joins, slots, kind = plan(lengths, key_lengths, heads, kv_heads, element_size, causal, _lib.ATTENTION_FORWARD)
    group, rows_per = heads // kv_heads, 32 if kind else 128
    # 256 compute units without a GPU
    tall = sum((n * group + 127) // 128 for n in lengths) * kv_heads
    assert bool(kind) == (max(lengths) * group <= 32 or (tall <= 128 and element_size == 4 and max(key_lengths) <= 128))
    spans, used = {}, []
    for qs, ql, ks, kl, row0, begin, end, slot in items:
        spans.setdefault((qs, ql, ks, kl, row0), []).append((begin, end, slot))
        assert 0 <= begin <= max(end, 0) and end <= kl and row0 % rows_per == 0 and row0 < ql * group
        if slot >= 0:
            used.append(slot)
    assert sorted(used) == list(range(slots))
    joined = {tuple(j[:5]): (j[5], j[7]) for j in joins}
    assert len(joined) == len(joins)
    a = b = 0
    for n, m in zip(lengths, key_lengths):
        for row0 in range(0, n * group, rows_per):
            parts = sorted(spans.pop((a, n, b, m, row0)))
            last = (min(n * group, row0 + rows_per) - 1) // group
            end = max(0, min(m, last + m - n + 1)) if causal else m
            assert parts[0][0] == 0 and parts[-1][1] == end
            assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
            if len(parts) == 1:
                assert parts[0][2] == -1
            else:
                n_parts, first = joined[(a, n, b, m, row0)]
                assert sorted(p[2] for p in parts) == list(range(first, first + n_parts))
        a, b = a + n, b + m
    assert not spans
    if kind == 2:                       # one turn each: no item has more tiles of 32 keys than there are wavefronts
        assert all(end - begin <= 4 * 32 for _, _, _, _, _, begin, end, _ in items)


@pytest.mark.parametrize("lengths, key_lengths, heads, kv_heads", CASES)
@pytest.mark.parametrize("causal", [False, True])
def test_key_items_cover_every_key_and_every_query_that_sees_it(lengths, key_lengths, heads, kv_heads, causal):
    items, joins, slots, kind = plan(lengths, key_lengths, heads, kv_heads, 2, causal, _lib.ATTENTION_GRAD_KEYS)
    group = heads // kv_heads
    tall = sum((m + 127) // 128 for m in key_lengths) * kv_heads
    parts = max(1, min(group, 512 // tall))                      # 256 compute units without a GPU
    assert len(joins) == (len(items) // parts if parts > 1 else 0) and slots == (len(items) if parts > 1 else 0)
    seen = {}
    for qs, ql, ks, kl, key0, begin, end, slot in items:
        first = max(0, key0 - (kl - ql)) if causal else 0       # the first query that sees the tile's first key
        assert begin <= first and 0 <= begin and end == ql
        seen.setdefault((ks, kl, key0), []).append(slot)
    for j in joins:
        assert j[5] == parts and j[7] % parts == 0 and sorted(seen[j[2], j[3], j[4]]) == list(range(j[7], j[7] + parts))
    if parts == 1:
        assert all(v == [-1] for v in seen.values())
    b = 0
    want = set()
    for m in key_lengths:
        want |= {(b, m, key0) for key0 in range(0, m, 32 if kind else 128)}
        b += m
    assert set(seen) == want


def test_items_are_laid_down_longest_first():
    items, _, _, _ = plan([3000, 10, 500], [3000, 10, 500], 4, 4, 2, True, _lib.ATTENTION_GRAD_QUERIES)
    spans = [i[6] - i[5] for i in items]
    assert spans == sorted(spans, reverse=True)


def test_plan_refuses_what_it_cannot_lay_down():
    L = _lib.lib
    one, counts = (ctypes.c_int * 1)(4), (ctypes.c_longlong * 4)()
    p, c = ctypes.addressof(one), ctypes.addressof(counts)
    ok = lambda *a: L.faith_attention_plan(*a)
    assert ok(None, p, 1, 4, 4, 2, 64, 0, 0, None, 0, c) == -1
    assert ok(p, p, 0, 4, 4, 2, 64, 0, 0, None, 0, c) == -2
    assert ok(p, p, 1, 4, 3, 2, 64, 0, 0, None, 0, c) == -2
    assert ok(p, p, 1, 4, 4, 3, 64, 0, 0, None, 0, c) == -3
    assert ok(p, p, 1, 4, 4, 2, 64, 0, 9, None, 0, c) == -3
    assert ok(p, p, 1, 4, 4, 2, 129, 0, 0, None, 0, c) == -3
    one[0] = -1
    assert ok(p, p, 1, 4, 4, 2, 64, 0, 0, None, 0, c) == -2
    one[0] = 400
    room = (ctypes.c_int * 8)()          # one item; 400 rows of each of four heads are more
    assert ok(p, p, 1, 4, 4, 2, 64, 0, 0, ctypes.addressof(room), 1, c) == -2 and b"room" in L.faith_last_error()


def test_entry_points_check_on_the_host():
    """Misaligned, overlapping, missing: a status, before anything is launched."""
    L = _lib.lib
    buf = (ctypes.c_float * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def forward_call(q=p, k=p, v=p, out=p, items=p, n=1, ts=64, hs=16, heads=4, kv_heads=4, size=16, dtype=0, scale=0.5, joins=0, kind=0):
        return L.faith_attention(q, k, v, out, None, None, items, n, joins, kind, ts, hs, ts, hs, ts, hs, ts, hs, 4, heads, kv_heads, size,
                                 dtype, 0, scale, None)
    assert forward_call(n=0) == 0
    assert forward_call(q=None) == -1 and forward_call(items=None) == -1 and forward_call(joins=1) == -1
    assert forward_call(k=None) == -4 and forward_call(q=p + 4) == -4 and forward_call(ts=8) == -4 and forward_call(hs=2) == -4 and forward_call(ts=1 << 22) == -4
    assert forward_call(size=18) == -3 and forward_call(size=132) == -3 and forward_call(size=4, dtype=1) == -3
    assert forward_call(dtype=3) == -3 and forward_call(kind=3) == -3 and forward_call(scale=0.0) == -3 and forward_call(scale=math.nan) == -3
    assert forward_call(kv_heads=3) == -2
    assert forward_call(n=1 << 27) == -3
    strides = (ctypes.c_longlong * 16)(*[64, 16] * 8)

    def backward_call(t=p, lse=p, stat=p, n=1, s=ctypes.addressof(strides), size=16, scale=0.5, kind=1, joins=0):
        return L.faith_attention_backward(t, t, t, t, t, lse, t, t, t, stat, None, p, n, kind, p, n, joins, 0, 0, s, 4, 4, 4, size, 0, 0, scale, None)
    assert backward_call(n=0) == 0
    assert backward_call(t=None) == -1 and backward_call(lse=None) == -1 and backward_call(stat=None) == -1 and backward_call(s=None) == -1
    assert backward_call(t=p + 4) == -4 and backward_call(size=130) == -3 and backward_call(scale=-1.0) == -3 and backward_call(kind=4) == -3
    assert backward_call(joins=-1) == -2 and backward_call(joins=2) == -2

    def norm_call(x=p, y=p, rows=1, n=8, kind=0, dtype=0, bits=0, scales=p, eps=1e-6):
        return L.faith_residual_norm(x, None, None, None, y, None, None, scales, rows, n, kind, dtype, bits, eps, None)
    assert norm_call(rows=0) == 0
    assert norm_call(x=None) == -1 and norm_call(y=None) == -1 and norm_call(bits=1, scales=None) == -1
    assert norm_call(n=0) == -2 and norm_call(rows=-1) == -2 and norm_call(rows=1 << 24) == -3
    assert norm_call(kind=3) == -3 and norm_call(dtype=5) == -3 and norm_call(bits=3) == -3 and norm_call(eps=-1.0) == -3 and norm_call(eps=math.nan) == -3
    assert L.faith_residual_norm_backward(p, None, p, None, p, p, p, None, None, 1, 8, 0, 0, None) == -1
    assert L.faith_residual_norm_backward(p, None, p, None, None, p, None, None, None, 1, 8, 0, 0, None) == -1
    assert L.faith_residual_norm_backward(p, None, p, None, p, p, None, None, None, 1, 8, 7, 0, None) == -3


@pytest.mark.parametrize("lengths, keys, what", [([], None, "no sequences"), ([3, -1], None, "not a length"), ([2.5], None, "not a length"),
                                                 ([True], None, "not a length"), ([3], [3, 3], "1 sequences of queries, 2 of keys"),
                                                 ([1 << 30], None, "not a length"), ([(1 << 30) - 1] * 3, None, "2\\^31")])
def test_packing_checks_lengths(lengths, keys, what):
    with pytest.raises(ValueError, match=what):
        ops.Packing(lengths, keys)


def test_packing_lives_on_the_gpu():
    with pytest.raises(ValueError, match="no CPU path"):
        ops.Packing([3], device="cpu")
    assert ops.Packing(torch.tensor([3, 0, 2])).starts() == [0, 3, 3, 5]


def test_operators_refuse_cpu_tensors_and_other_types():
    packing = ops.Packing([3])
    q = torch.zeros(3, 2, 16)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.attention(q, q, q, packing)
    with pytest.raises(TypeError, match="Packing"):
        ops.attention(q, q, q, [3])
    with pytest.raises(TypeError, match="tensor"):
        ops.attention(None, q, q, packing)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.residual_norm(torch.zeros(3, 16))
    with pytest.raises(TypeError, match="tensor"):
        ops.residual_norm([1.0])
    with pytest.raises(ValueError, match="no CPU path"):
        ops.residual_norm_backward(torch.zeros(3, 16), torch.zeros(3, 16), None, torch.zeros(3))


def test_concrete_checks_embeddings_and_positions():
    with pytest.raises(ValueError, match="embeddings"):
        concrete._rows_of(torch.zeros(3, 4), None)
    with pytest.raises(ValueError, match="embeddings"):
        concrete._rows_of(torch.zeros(2, 3, 4), [3, 3])
    with pytest.raises(ValueError, match="2 positions, 1 radii"):
        concrete.falsify(None, torch.zeros(1, 4, 8), [1, 2], [0.1], 0)
    with pytest.raises(ValueError, match="outside"):
        concrete.falsify(None, torch.zeros(1, 4, 8), [4], [0.1], 0)
    assert concrete.falsify(None, torch.zeros(1, 4, 8), [], [], 0) == []
    from types import SimpleNamespace
    net = SimpleNamespace(classifier=SimpleNamespace(weight=torch.zeros(2, 8)))
    emb = torch.zeros(1, 4, 8)
    for bad, what in ((dict(label=2), "classes"), (dict(label=-1), "classes"), (dict(label=0.5), "classes"), (dict(p=0.5), "norm"), (dict(steps=-1), "steps"),
                      (dict(radii=[-0.1]), "radius"), (dict(radii=[math.nan]), "radius"), (dict(radii=[math.inf]), "radius"), (dict(p=math.nan), "norm")):
        args = dict(radii=[0.1], label=0)
        args.update(bad)
        with pytest.raises(ValueError, match=what):
            concrete.falsify(net, emb, [1], **args)
    net.classifier.weight = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="two classes"):
        forward.verify_safety(None, net, emb, 1, 0.1, None)


@pytest.mark.parametrize("p", [1.0, 1.5, 2.0, 3.0, math.inf])
def test_steps_of_the_search_stay_in_the_ball_and_ascend(p):
    g = torch.Generator().manual_seed(5)
    x, r = torch.randn(6, 9, generator=g), torch.tensor([0.1, 0.5, 1.0, 2.0, 0.0, 3.0])
    d = concrete._steepest(x, p)
    norm = lambda t: torch.linalg.vector_norm(t, ord=p, dim=1)
    assert torch.allclose(norm(d), torch.ones(6), rtol=1e-5)
    # no direction of unit norm grows a linear function faster than its dual norm says
    q = math.inf if p == 1 else 1.0 if math.isinf(p) else p / (p - 1)
    assert torch.allclose((x * d).sum(1), torch.linalg.vector_norm(x, ord=q, dim=1), rtol=1e-5)
    inside = concrete._into_ball(x, p, r)
    assert bool((norm(inside) <= r * (1 + 1e-5)).all())


def test_bounds_of_what_only_the_concrete_pass_knows_are_refused():
    from types import SimpleNamespace
    from faith_amd.workloads import random_layer
    g = torch.Generator().manual_seed(3)
    net = SimpleNamespace(embedding_norm=None, layers=[random_layer(g, 16, 4, 32)], layer_norm="no_var", hidden_act="relu")
    forward._bounded(net)
    net.causal = True
    with pytest.raises(ValueError, match="causal"):
        forward.propagate(None, net)
    net.causal, net.layer_norm = False, "rms"
    with pytest.raises(ValueError, match="rms"):
        forward.propagate(None, net)
    net.layer_norm = "standard"
    net.layers[0].attention.self.num_key_value_heads = 2
    with pytest.raises(ValueError, match="share"):
        forward.propagate(None, net)


def test_random_lengths_give_items_within_the_sequences():
    rng = random.Random(8)
    for _ in range(60):
        n = rng.randint(1, 9)
        ql = [rng.choice([0, 1, rng.randint(0, 400)]) for _ in range(n)]
        kl = [rng.choice([0, 1, rng.randint(0, 900)]) for _ in range(n)]
        kv = rng.choice([1, 2, 8])
        for which in range(3):
            items, joins, slots, kind = plan(ql, kl, kv * rng.choice([1, 3, 4]), kv, rng.choice([2, 4]), rng.random() < 0.5, which)
            for qs, a, ks, b, row0, begin, end, slot in items:
                i = next(i for i in range(n) if sum(ql[:i]) == qs and sum(kl[:i]) == ks and (ql[i], kl[i]) == (a, b))
                assert 0 <= begin and end <= (b if which < 2 else a) and slot < max(1, slots), i


def test_results_whose_heads_share_memory_are_refused():
    """Heads that lie on each other may be read (one key head seen as many); written, they would race."""
    L = _lib.lib
    buf = (ctypes.c_float * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def forward_call(hs, heads=4):
        return L.faith_attention(p, p, p, p, None, None, p, 1 << 27, 0, 0, 64, 0, 64, 0, 64, 0, 64, hs, 4, heads, heads, 16, 0, 0, 0.5, None)
    assert forward_call(0) == -4 and forward_call(12) == -4
    # past this check, and refused for its number of items: nothing is launched
    assert forward_call(16) == -3 and forward_call(0, heads=1) == -3

    def backward_call(which):
        strides = (ctypes.c_longlong * 16)(*[64, 16] * 8)
        strides[2 * which + 1] = 0
        return L.faith_attention_backward(p, p, p, p, p, p, p, p, p, p, None, p, 1 << 27, 0, p, 1 << 27, 0, 0, 0, ctypes.addressof(strides), 4, 4, 4, 16, 0, 0, 0.5, None)
    assert [backward_call(i) for i in range(8)] == [-3] * 5 + [-4] * 3


def test_what_is_kept_of_a_call_holds_no_number_of_it():
    from types import SimpleNamespace
    q = torch.zeros(4, 2, 16)
    packing = SimpleNamespace(device=SimpleNamespace(index=q.get_device()), _calls={})
    key, _ = ops._known_call(packing, 0, True, q, q, q)
    assert key is not None and not any(isinstance(x, (torch.Tensor, float)) for x in key)


def test_a_scale_that_asks_for_a_gradient_is_refused():
    q = torch.zeros(4, 2, 16)
    with pytest.raises(ValueError, match="scale"):
        concrete.attention(q, q, q, ops.Packing([4]), scale=torch.tensor(0.5, requires_grad=True))


def norm_of(d, p):
    return torch.linalg.vector_norm(d.double(), ord=math.inf if p >= 10 else p, dim=1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("p", [1.0, 1.5, 2.0, math.inf])
@pytest.mark.parametrize("radius", [1e-6, 1e-3, 1e-2, 0.05, 3.0])
def test_the_perturbation_that_the_network_sees_is_in_the_ball(dtype, p, radius):
    """Rounded to the embeddings' type, at radii far under, near and far over one step of it; zeros and the largest values too."""
    g = torch.Generator().manual_seed(17)
    base = torch.randn(40, 256, generator=g).to(dtype)
    base[0], base[1, ::2], base[2, ::3] = 0, 0, torch.finfo(dtype).max
    base[3] = torch.finfo(dtype).tiny
    r = torch.full((40,), radius, dtype=torch.float64)
    for d in (torch.randn(40, 256, generator=g), concrete._steepest(torch.randn(40, 256, generator=g), p)):
        delta = concrete._into_ball(d.double() * radius, p, r)
        moved = concrete._moved(base, delta)
        assert moved.dtype == dtype and bool(torch.isfinite(moved).all())
        assert bool((norm_of(moved.double() - base.double(), p) <= r).all())
        # and no further in than one step of the type: eps of a magnitude that |base| + |delta| bounds
        ulp = (base.double().abs() + delta.abs()) * torch.finfo(dtype).eps + torch.finfo(dtype).smallest_normal
        short = (moved.double() - base.double() - delta).abs()
        assert bool((short[3:] <= ulp[3:]).all())


def searched(monkeypatch, logits, embeddings, radii, p=2.0, steps=4, label=0):
    """falsify on the CPU, on a network that is one function of its rows; also every perturbation that it looked at."""
    from types import SimpleNamespace
    n, length = len(radii), embeddings.shape[1]
    seen = []

    def run(network, x, batch, activations=None):
        rows = x.view(n, length, -1)
        seen.append((rows.detach() - 0)[:, 1].double() - embeddings[0, 1].double())
        return logits(rows)
    monkeypatch.setattr(concrete, "_logits", run)
    net = SimpleNamespace(classifier=SimpleNamespace(weight=torch.zeros(2, embeddings.shape[2])))
    batch = SimpleNamespace(packing=SimpleNamespace(lengths=(length,) * n), first=torch.arange(n) * length)
    return concrete.falsify(net, embeddings, [1] * n, radii, label, p, steps, batch), seen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_the_search_stays_in_the_ball(monkeypatch, dtype, p):
    g = torch.Generator().manual_seed(3)
    emb, w = torch.randn(1, 3, 256, generator=g).to(dtype), torch.randn(2, 256, generator=g)
    radii = [0.0, 1e-4, 1e-3, 0.01, 0.05, 0.1, 1.0, 30.0]
    found, seen = searched(monkeypatch, lambda rows: torch.tanh(rows[:, 1].float() @ w.t() / 16), emb, radii, p, label=int((emb[0, 1].float() @ w.t()).argmax()))
    assert len(seen) == 5
    for moved in seen:
        assert bool((norm_of(moved, p) <= torch.tensor(radii, dtype=torch.float64)).all())
    assert found[-1] and not found[0]


def test_what_is_no_number_proves_nothing(monkeypatch):
    emb = torch.ones(1, 3, 4)
    column = lambda m: torch.stack([m, torch.zeros_like(m)], 1)
    # a margin that is NaN everywhere, one that becomes NaN or infinite away from the sentence
    for f in (lambda x: x[:, 1, 0] * math.nan, lambda x: torch.sqrt(x[:, 1, 0] - 0.999999), lambda x: 1 / (x[:, 1, 0] - 0.5).clamp_min(0) * 0 + 1,
              lambda x: torch.where(x[:, 1, 0] < 1, -math.inf, 1.0) + 0 * x[:, 1, 0]):
        found, _ = searched(monkeypatch, lambda rows: column(f(rows)), emb, [0.5, 0.6])
        assert found == [False, False]

    class Overflow(torch.autograd.Function):
        """A margin of one whose gradient is infinite and NaN."""
        @staticmethod
        def forward(ctx, x):
            return torch.ones(x.shape[0])

        @staticmethod
        def backward(ctx, g):
            bad = torch.full((2, 3, 4), math.inf)
            bad[1, 1, 2] = math.nan
            return bad
    found, seen = searched(monkeypatch, lambda rows: column(Overflow.apply(rows)), emb, [0.5, 0.6])
    assert found == [False, False] and all(bool((d == 0).all()) for d in seen)


def test_the_search_takes_one_sentence():
    from types import SimpleNamespace
    net = SimpleNamespace(classifier=SimpleNamespace(weight=torch.zeros(2, 8)))
    for shape in ((2, 4, 8), (4, 8), (0, 4, 8)):
        with pytest.raises(ValueError, match="one sentence"):
            concrete.falsify(net, torch.zeros(shape), [1, 2], [0.1, 0.1], 0)


def test_rows_of_the_norm_that_pass_one_launch_are_refused():
    """Before anything is launched: 2^32 threads, which rows of eight wavefronts reach at half as many."""
    L = _lib.lib
    buf = (ctypes.c_float * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(rows, n, dtype):
        return L.faith_residual_norm(p, None, None, None, p, None, None, p, rows, n, 0, dtype, 0, 1e-6, None)
    for n, dtype in ((8192, _lib.BF16), (16384, _lib.F16), (8192, _lib.F32), (4096, _lib.F32)):
        assert call(1 << 23, n, dtype) == -3 and b"launch" in L.faith_last_error()
    for n, dtype in ((64, _lib.BF16), (4096, _lib.BF16), (2048, _lib.F32), (7, _lib.F32), (40000, _lib.F32)):
        assert call(1 << 24, n, dtype) == -3 and b"launch" in L.faith_last_error()


def test_rows_of_the_norm_longer_than_its_counters_are_refused():
    L = _lib.lib
    buf = (ctypes.c_float * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    for n in ((1 << 30) + 1, (1 << 31) - 1, (1 << 31) - 256):
        assert L.faith_residual_norm(p, None, None, None, p, None, None, p, 1, n, 0, 0, 0, 1e-6, None) == -2
        assert L.faith_residual_norm_backward(p, None, p, None, p, p, None, None, None, 1, n, 0, 0, None) == -2


def test_results_whose_rows_share_memory_with_other_heads_are_refused():
    """Token by token or head by head; what lies in between is written by two workgroups."""
    L = _lib.lib
    buf = (ctypes.c_float * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def forward_call(ts, hs, heads=4):          # refused (-3) for its number of items where the strides pass
        return L.faith_attention(p, p, p, p, None, None, p, 1 << 27, 0, 0, 64, 16, 64, 16, 64, 16, ts, hs, 4, heads, heads, 16, 0, 0, 0.5, None)
    for ts, hs in ((16, 16), (32, 16), (60, 16), (24, 32), (64, 20)):
        assert forward_call(ts, hs) == -4 and b"overlap" in L.faith_last_error()
    for ts, hs in ((64, 16), (76, 20), (16, 32), (16, 1000), (24, 40)):
        assert forward_call(ts, hs) == -3
    assert forward_call(16, 16, heads=1) == -3

    def backward_call(which, ts, hs):
        strides = (ctypes.c_longlong * 16)(*[64, 16] * 8)
        strides[2 * which], strides[2 * which + 1] = ts, hs
        return L.faith_attention_backward(p, p, p, p, p, p, p, p, p, p, None, p, 1 << 27, 0, p, 1 << 27, 0, 0, 0, ctypes.addressof(strides), 4, 4, 4, 16, 0, 0, 0.5, None)
    assert [backward_call(i, 16, 16) for i in range(8)] == [-3] * 5 + [-4] * 3
    assert [backward_call(i, 16, 640) for i in range(8)] == [-3] * 8


@pytest.mark.parametrize("hs", [0, 32, 40, 63, 64, 4096, 1 << 24])
def test_the_stride_of_a_single_token_passes_for_two(hs):
    ts = ops._stride_of_one(hs, 4, 32)
    assert hs < 32 or ts >= 3 * hs + 32 or hs >= ts + 32
    assert ts < 1 << 22


def test_arrays_in_lds_are_aligned_for_their_widest_read():
    """16 bytes a lane: not left to where the compiler puts an array of 2-byte elements."""
    import glob
    import os
    import re
    import faith_amd
    folder = os.path.join(os.path.dirname(faith_amd.__file__), "csrc")
    seen = 0
    for path in [p for name in ("attention", "residual_norm") for p in glob.glob(os.path.join(folder, name + "*"))]:
        for line in open(path):
            if re.search(r"\b__shared__\b", line) and "[" in line:
                seen += 1
                assert "__align__(16)" in line, f"{os.path.basename(path)}: {line.strip()}"
    assert seen >= 8


def test_the_device_guard_asks_for_the_current_device(monkeypatch):
    """By the public name: every operator of the library goes through it."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    assert ops._on(torch.device("cuda", 1)) is ops._NO_GUARD and ops._on(torch.device("cuda")) is ops._NO_GUARD
    other = ops._on(torch.device("cuda", 0))
    assert isinstance(other, torch.cuda.device) and other.idx == 0


def test_networks_that_say_none_for_shared_key_heads_have_their_own():
    """None is what a configuration without them holds: such a network was propagated before there was an attribute to look at."""
    from types import SimpleNamespace
    from faith_amd.workloads import random_layer
    net = SimpleNamespace(embedding_norm=None, layers=[random_layer(torch.Generator().manual_seed(3), 16, 4, 32)], layer_norm="no_var", hidden_act="relu")
    net.layers[0].attention.self.num_key_value_heads = None
    forward._bounded(net)
    net.layers[0].attention.self.num_key_value_heads = 4
    forward._bounded(net)


@pytest.mark.parametrize("mode", ["no", "standard"])
def test_activations_of_another_name_are_refused_whatever_the_network_normalises(mode):
    from types import SimpleNamespace
    net = SimpleNamespace(layer_norm=mode)
    for ask in (concrete.logits, concrete.predict):
        with pytest.raises(ValueError, match="activations"):
            ask(net, torch.zeros(1, 3, 8), activations="int4")
