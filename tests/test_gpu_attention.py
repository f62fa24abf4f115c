"""Attention of the concrete pass and its gradients against the definition in float64 (tests/concrete_reference.py, which also
derives how far roundings may carry a result)."""
import math

import pytest
import torch

from tests import concrete_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [  # lengths, key lengths (None: alike), heads, key heads, causal
    ([5, 1, 33], None, 4, 2, True),
    ([32] * 3, None, 4, 4, False),
    ([128, 65, 200], None, 6, 2, True),
    ([1, 1, 1], [700, 3, 65], 8, 2, True),
    ([1, 4], [3000, 20], 4, 4, False),
    ([130, 0, 7], [300, 5, 0], 2, 1, True),       # no queries; no keys
    ([40, 9], [10, 9], 3, 1, True),               # the first 30 queries see nothing
    ([70], [5000], 4, 2, False),
    ([1], [1], 1, 1, True),
    ([31, 64, 129], [63, 64, 127], 2, 2, False),
    ([200, 33], None, 10, 2, True),               # gradients of keys in parts of the group
    ([2100, 1500], None, 6, 3, True),
    ([300] * 40, None, 4, 4, False),              # workgroups of 128 rows in every pass
]


def tensors(lengths, keys, heads, kv_heads, size, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda t, h: (torch.randn(t, h, size, generator=g, device="cuda") * scale).to(dtype)
    return rnd(sum(lengths), heads), rnd(sum(keys), kv_heads), rnd(sum(keys), kv_heads), rnd(sum(lengths), heads)


@pytest.mark.parametrize("dtype, size", [(F32, 64), (F32, 4), (F32, 32), (F32, 100), (F32, 128), (BF16, 8), (BF16, 32), (BF16, 64), (BF16, 80),
                                         (BF16, 128), (F16, 64), (F16, 96), (F16, 128)])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_and_gradients(case, dtype, size):
    from faith_amd import ops
    lengths, keys, heads, kv_heads, causal = SHAPES[case]
    keys = keys or lengths
    q, k, v, dout = tensors(lengths, keys, heads, kv_heads, size, dtype, seed=case)
    packing = ops.Packing(lengths, keys)
    out, lse = ops.attention(q, k, v, packing, causal=causal, return_lse=True)
    grads = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=causal)
    r = R.attention(q, k, v, lengths, keys, causal, 1 / math.sqrt(size), dout)
    R.check("out", out, r["out"], r["out_tol"])
    assert bool((torch.isinf(lse) == torch.isinf(r["lse"])).all())
    R.check("lse", lse, r["lse"], r["lse_tol"] + 1e-30)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert got.dtype == dtype
        R.check(name, got, r[name], r[name + "_tol"])
    # without the logarithms: the same result; the same call: the same bits
    assert torch.equal(out, ops.attention(q, k, v, packing, causal=causal))
    again = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale, spread", [(0.3, 1.0), (1.0, 6.0), (4.0, 0.01)])
def test_scores_far_apart_and_other_scales(dtype, scale, spread):
    """Large scores: the running reference moves many times.  (Scores of hundreds: a probability's error grows with them,
    and the tolerance with it.)"""
    from faith_amd import ops
    lengths = [300, 77]
    q, k, v, dout = tensors(lengths, lengths, 2, 1, 64, dtype, 3, 1.0)
    q = (q.float() * spread).to(dtype)
    k = (k.float() * torch.linspace(0.1, 1, k.shape[0], device="cuda")[:, None, None]).to(dtype)      # later keys larger: later maxima
    packing = ops.Packing(lengths)
    out, lse = ops.attention(q, k, v, packing, causal=True, scale=scale, return_lse=True)
    grads = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=True, scale=scale)
    r = R.attention(q, k, v, lengths, lengths, True, scale, dout)
    R.check("out", out, r["out"], r["out_tol"])
    for name, got in zip(("dq", "dk", "dv"), grads):
        R.check(name, got, r[name], r[name + "_tol"])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_views_of_one_projection_and_other_layouts(dtype):
    """q, k, v as slices of one [tokens, (heads + 2 key heads) * size] array; heads in front; a result that the caller brings,
    inside a larger array whose other places stay as they were."""
    from faith_amd import ops
    lengths, heads, kv_heads, size = [37, 90], 4, 2, 32
    g = torch.Generator(device="cuda").manual_seed(1)
    t = sum(lengths)
    both = torch.randn(t + 3, (heads + 2 * kv_heads) * size, generator=g, device="cuda").to(dtype)
    both[t:] = math.nan                                                    # rows behind the last sequence
    q, k, v = both.view(t + 3, -1, size).split([heads, kv_heads, kv_heads], 1)
    packing = ops.Packing(lengths)
    want = ops.attention(q[:t].contiguous(), k[:t].contiguous(), v[:t].contiguous(), packing, causal=True)
    got, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
    assert torch.equal(got[:t], want) and bool((got[t:] == 0).all())
    large = torch.full((t + 5, heads + 1, size), 7.0, device="cuda", dtype=dtype)
    ops.attention(q, k, v, packing, causal=True, out=large[2:, 1:])
    assert torch.equal(large[2:t + 2, 1:], want)
    assert bool((large[:2] == 7).all()) and bool((large[t + 2:] == 7).all()) and bool((large[:, 0] == 7).all())
    front = lambda x: x[:t].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.attention(front(q), front(k), front(v), packing, causal=True), want)
    dout = torch.randn(t, heads, size, generator=g, device="cuda").to(dtype)
    a = ops.attention_backward(front(dout), q, k, v, got, lse, packing, causal=True)
    b = ops.attention_backward(dout, q[:t].contiguous(), k[:t].contiguous(), v[:t].contiguous(), want, lse, packing, causal=True)
    assert all(torch.equal(x[:t], y) and bool((x[t:] == 0).all()) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lengths, keys", [([50], [50]), ([3], [400]), ([200], [200]), ([2], [3000])])
def test_masked_places_may_hold_anything(dtype, bad, lengths, keys):
    """NaN or infinity in the last key and value: every query but the last is masked from it.  In the first query and its
    gradient: every key behind the first that it sees is masked from it."""
    from faith_amd import ops
    q, k, v, dout = tensors(lengths, keys, 2, 1, 64, dtype, 9)
    n, packing = lengths[0], ops.Packing(lengths, keys)
    scale = 1 / math.sqrt(64)
    k0, v0 = k.clone(), v.clone()
    k0[-1], v0[-1] = 0, 0
    k[-1, :, 5], v[-1, :, 7] = bad, bad
    r = R.attention(q, k0, v0, lengths, keys, True, scale, dout)
    out, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
    R.check("out", out[:n - 1], r["out"][:n - 1], r["out_tol"][:n - 1])
    dq, _, _ = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=True)
    R.check("dq", dq[:n - 1], r["dq"][:n - 1], r["dq_tol"][:n - 1])
    # and the other way round
    q, k, v, dout = tensors(lengths, keys, 2, 1, 64, dtype, 10)
    q0, dout0 = q.clone(), dout.clone()
    q0[0], dout0[0] = 0, 0
    q[0, :, 3], dout[0, :, 2] = bad, bad
    out, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
    _, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=True)
    r = R.attention(q0, k, v, lengths, keys, True, scale, dout0)
    seen = keys[0] - n + 1                                                  # keys that the first query sees
    R.check("dk", dk[seen:], r["dk"][seen:], r["dk_tol"][seen:])
    R.check("dv", dv[seen:], r["dv"][seen:], r["dv_tol"][seen:])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lengths, keys, causal", [([1] * 9, [1] * 9, False), ([1, 1], [1, 1], True), ([70, 300], [1, 1], False), ([40, 5], [40, 5], True), ([5], [3], True)])
def test_a_query_that_sees_one_key_has_no_gradient_through_its_score(dtype, lengths, keys, causal):
    """Its probability is 1 whatever the score: dq is zero, and it adds nothing to dk, not merely little."""
    from faith_amd import ops
    q, k, v, dout = tensors(lengths, keys, 4, 2, 64, dtype, 12)
    packing = ops.Packing(lengths, keys)
    out, lse = ops.attention(q, k, v, packing, causal=causal, return_lse=True)
    dq, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=causal)
    r = R.attention(q, k, v, lengths, keys, causal, 0.125, dout)
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        R.check(name, got, r[name], r[name + "_tol"])
    a = 0
    for n, m in zip(lengths, keys):
        i = m_only = max(0, n - m)                               # the first query that sees a key
        alone = dq[a:a + n] if m == 1 else dq[a + i:a + i + 1] if causal else dq[:0]
        assert bool((alone == 0).all()), m_only
        a += n
    if max(keys) == 1:
        assert bool((dk == 0).all())


def test_not_a_number_where_it_is_seen_stays_one():
    from faith_amd import ops
    q, k, v, _ = tensors([40], [40], 1, 1, 32, BF16, 2)
    v[17, 0, 3] = math.nan
    out = ops.attention(q, k, v, ops.Packing([40]), causal=True)
    assert bool(torch.isnan(out[17:, 0, 3]).all()) and not bool(torch.isnan(out[:17]).any())
    assert not bool(torch.isnan(out[:, 0, :3]).any()) and not bool(torch.isnan(out[:, 0, 4:]).any())


@pytest.mark.parametrize("kv_heads, heads, lengths, keys", [(8, 32, [1] * 5, [8192, 1, 513, 4000, 257]), (1, 1, [1], [20000]), (2, 16, [2, 1], [3000, 300]),
                                                            (1, 1, [32], [7000]), (1, 4, [128], [9000])])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_rows_against_many_keys(kv_heads, heads, lengths, keys, dtype):
    """Keys cut into parts and joined."""
    from faith_amd import _lib, ops
    q, k, v, _ = tensors(lengths, keys, heads, kv_heads, 128, dtype, 4)
    packing = ops.Packing(lengths, keys)
    assert packing.plan(_lib.ATTENTION_FORWARD, heads, kv_heads, q.element_size(), 128, True)[3] > 0
    out, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
    r = R.attention(q, k, v, lengths, keys, True, 1 / math.sqrt(128))
    R.check("out", out, r["out"], r["out_tol"])
    R.check("lse", lse, r["lse"], r["lse_tol"])


def test_offsets_past_32_bits():
    """A cache whose last sequence starts 4.3 GB into the array."""
    from faith_amd import ops
    skip, heads, size = (1 << 32) // (8 * 128 * 2) + 1000, 8, 128
    k = torch.empty(skip + 300, heads, size, device="cuda", dtype=BF16)
    v = torch.empty_like(k)
    g = torch.Generator(device="cuda").manual_seed(2)
    k[skip:] = torch.randn(300, heads, size, generator=g, device="cuda").to(BF16)
    v[skip:] = torch.randn(300, heads, size, generator=g, device="cuda").to(BF16)
    q = torch.randn(200, heads, size, generator=g, device="cuda").to(BF16)
    for n in (1, 200):
        got = ops.attention(q[:n], k, v, ops.Packing([0, n], [skip, 300]), causal=True)
        want = ops.attention(q[:n], k[skip:], v[skip:], ops.Packing([n], [300]), causal=True)
        assert torch.equal(got, want)


def test_gradients_against_differences():
    """Along random directions, central differences of the definition in float64: the error of a difference of step h is
    h^2 / 6 times a third derivative (of order one here) plus rounding of 1e-16 / h."""
    from faith_amd import ops
    lengths, heads, kv_heads, size = [13, 30], 4, 2, 16
    q, k, v, dout = tensors(lengths, lengths, heads, kv_heads, size, F32, 6)
    packing = ops.Packing(lengths)
    out, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
    grads = ops.attention_backward(dout, q, k, v, out, lse, packing, causal=True)

    def loss(*x):
        total, a = 0.0, 0
        for n in lengths:
            for h in range(heads):
                qs, ks, vs = x[0][a:a + n, h], x[1][a:a + n, h // 2], x[2][a:a + n, h // 2]
                s = (qs @ ks.t() / math.sqrt(size)).masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
                total = total + (torch.softmax(s, 1) @ vs * dout[a:a + n, h].double()).sum()
            a += n
        return total
    g = torch.Generator(device="cuda").manual_seed(7)
    base, h = [t.double() for t in (q, k, v)], 1e-4
    for i in range(3):
        d = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
        d /= d.norm()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        want = float(loss(*up) - loss(*down)) / (2 * h)
        # the gradient's own error: some 1e-6 of its norm, along a unit direction
        assert abs(float((grads[i].double() * d).sum()) - want) <= 1e-5 * float(grads[i].norm()) + 1e-6


def test_captured_and_replayed_between_eager_work():
    from faith_amd import ops
    lengths, keys = [60, 7, 200], [60, 900, 200]
    q, k, v, dout = tensors(lengths, keys, 4, 2, 64, BF16, 8)
    packing, one = ops.Packing(lengths, keys), ops.Packing([1] * 3, keys)

    def body():
        out, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
        return (out, *ops.attention_backward(dout, q, k, v, out, lse, packing, causal=True), ops.attention(q[:3], k, v, one))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    results = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            results.append(body())
    for i in range(4):
        q.copy_(torch.randn(q.shape, device="cuda").to(BF16))
        want = body()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(want, result)), i


def test_first_call_inside_a_capture_is_refused():
    from faith_amd import ops
    q, k, v, _ = tensors([8], [8], 2, 2, 32, F32)
    packing = ops.Packing([8])
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before the capture"):
            ops.attention(q, k, v, packing)


def test_on_another_stream_with_other_work_in_flight():
    from faith_amd import ops
    lengths = [500, 90]
    q, k, v, _ = tensors(lengths, lengths, 8, 2, 128, BF16, 5)
    packing = ops.Packing(lengths)
    want = ops.attention(q, k, v, packing, causal=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [ops.attention(q, k, v, packing, causal=True) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got)


def test_workspace_keeps_results_of_every_type():
    from faith_amd import ops
    lengths = [40, 3000]
    q, k, v, _ = tensors([1, 1], lengths, 8, 2, 128, F16, 5)
    packing, ws = ops.Packing([1, 1], lengths), ops.Workspace()
    want = ops.attention(q, k, v, packing)
    for _ in range(3):
        with ops.workspace(ws):
            got = ops.attention(q, k, v, packing)
            assert torch.equal(got, want)
    n = ws.allocations
    with ops.workspace(ws):
        ops.attention(q, k, v, packing)
    assert ws.allocations == n


def test_refusals():
    from faith_amd import _lib, ops
    lengths = [6, 10]
    q, k, v, dout = tensors(lengths, lengths, 4, 2, 32, BF16)
    packing = ops.Packing(lengths)
    call = lambda q=q, k=k, v=v, p=packing, **kw: ops.attention(q, k, v, p, **kw)
    for bad, kind, what in [(dict(k=k.float()), TypeError, "k:"), (dict(q=q.double()), TypeError, "q:"), (dict(q=q[:15]), ValueError, "q: expected shape"),
                            (dict(k=k[:, :, :16]), ValueError, "k: expected shape"), (dict(v=v[:, :1]), ValueError, "v: expected shape"),
                            (dict(q=q[:, :3]), ValueError, "share"), (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), ValueError, "contiguous"),
                            (dict(q=q[0]), ValueError, "q: expected shape"), (dict(k=k[:1].expand(16, 2, 32)), ValueError, "overlap"),
                            (dict(scale=0.0), ValueError, "scale"), (dict(scale=math.inf), ValueError, "scale"), (dict(scale=-1.0), ValueError, "scale"),
                            (dict(q=torch.zeros(16 * 128 + 1, device="cuda", dtype=BF16)[1:].view(16, 4, 32)), ValueError, "16 bytes")]:
        with pytest.raises(kind, match=what):
            call(**bad)
    wide = torch.zeros(16, 2, 136, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="up to 128"):
        call(q=wide, k=wide, v=wide)
    with pytest.raises(ValueError, match="up to 128"):
        call(q=wide[:, :, :20], k=wide[:, :, :20], v=wide[:, :, :20])
    out, lse = ops.attention(q, k, v, packing, return_lse=True)
    with pytest.raises(ValueError, match="lse"):
        ops.attention_backward(dout, q, k, v, out, lse[:, :5], packing)
    with pytest.raises(ValueError, match="dout"):
        ops.attention_backward(dout[:, :2], q, k, v, out, lse, packing)
    with pytest.raises(ValueError, match="out: expected"):
        ops.attention(q, k, v, packing, out=out[:9])
    assert issubclass(_lib.FaithError, RuntimeError)


def test_empty_batches():
    from faith_amd import ops
    q, k, v, dout = tensors([0, 0], [5, 0], 2, 2, 32, F32)
    packing = ops.Packing([0, 0], [5, 0])
    out, lse = ops.attention(q, k, v, packing, return_lse=True)
    assert out.shape == (0, 2, 32) and lse.shape == (2, 0)
    dq, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, packing)
    assert dq.shape == (0, 2, 32) and bool((dk == 0).all()) and bool((dv == 0).all())
    q, k, v, dout = tensors([4, 1], [0, 0], 2, 2, 32, F32)              # queries, and no keys at all
    packing = ops.Packing([4, 1], [0, 0])
    for causal in (False, True):
        out, lse = ops.attention(q, k, v, packing, causal, return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
        dq, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, packing, causal)
        assert bool((dq == 0).all()) and dk.shape == (0, 2, 32) and dv.shape == (0, 2, 32)


def test_results_that_lie_on_each_other_are_refused():
    from faith_amd import ops
    lengths = [6, 10]
    q, k, v, _ = tensors(lengths, lengths, 4, 2, 32, BF16)
    packing = ops.Packing(lengths)
    want = ops.attention(q, k, v, packing)
    store = torch.zeros(16 * 4 * 40, device="cuda", dtype=BF16)
    for strides in [(128, 0, 1), (32, 0, 1), (32, 32, 1), (64, 32, 1), (40, 480, 1)]:
        with pytest.raises(ValueError, match="must not overlap"):
            ops.attention(q, k, v, packing, out=store.as_strided((16, 4, 32), strides))
    assert not store.any()
    # token by token with room between the heads, and head by head
    for strides in [(160, 40, 1), (32, 512, 1), (40, 640, 1)]:
        out = store.as_strided((16, 4, 32), strides)
        assert ops.attention(q, k, v, packing, out=out) is out and torch.equal(out, want)
    one = ops.Packing([1])
    out = store[:160].as_strided((1, 4, 32), (160, 40, 1))
    assert torch.equal(ops.attention(q[:1], k[:1], v[:1], one, out=out), ops.attention(q[:1], k[:1], v[:1], one))


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_a_scale_or_mask_given_as_a_tensor_is_read_by_every_call(where):
    """What a tensor holds now counts, not what it held when a call like this one was made first."""
    from faith_amd import ops
    lengths = [20, 5]
    q, k, v, dout = tensors(lengths, lengths, 4, 2, 32, F32)
    packing, fresh = ops.Packing(lengths), lambda: ops.Packing(lengths)
    scale, causal = torch.full((), 0.5, device=where), torch.tensor(True, device=where)
    for number, mask in ((0.5, True), (2.0, True), (2.0, False), (0.125, False), (0.5, True)):
        scale.fill_(number)
        causal.fill_(mask)
        out, lse = ops.attention(q, k, v, packing, causal, scale, return_lse=True)
        want, want_lse = ops.attention(q, k, v, fresh(), mask, number, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        got = ops.attention_backward(dout, q, k, v, out, lse, packing, causal, scale)
        assert all(torch.equal(a, b) for a, b in zip(got, ops.attention_backward(dout, q, k, v, out, lse, fresh(), mask, number)))
    # a scale that changes with every call (a temperature, a trained one) leaves nothing behind
    known = len(packing._calls)
    for i in range(20):
        ops.attention(q, k, v, packing, True, 0.1 + i)
    assert len(packing._calls) == known


def test_the_gradient_takes_the_scale_of_its_forward_call():
    from faith_amd import concrete, ops
    lengths = [9, 30]
    q, k, v, dout = tensors(lengths, lengths, 4, 4, 32, F32, 2)
    q.requires_grad_(True)
    scale = torch.tensor(0.5)
    out = concrete.attention(q, k, v, ops.Packing(lengths), scale=scale)
    scale.fill_(4.0)
    (got,) = torch.autograd.grad(out, q, dout)
    (want,) = torch.autograd.grad(concrete.attention(q, k, v, ops.Packing(lengths), scale=0.5), q, dout)
    assert torch.equal(got, want)


def small_gradient_reference(q, k, v, dout, scale):
    """One sequence, every head seeing every key, in float64: (dq, dk, dv) and their tolerances.  Rounding ds and p to the operands'
    type is half a step of each, at any size of theirs: nothing is added for values under the type's normal range but half the
    smallest step of the result, where a result lies there."""
    ut, u32 = R.half_step(q.dtype), R.U32
    (n, heads, size), (m, kv_heads, _) = q.shape, k.shape
    smallest = 2.0 ** -25
    grads = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
    tols = [torch.full_like(g, smallest) for g in grads]
    for h in range(heads):
        g = h // (heads // kv_heads)
        qh, kh, vh, do = q[:, h].double(), k[:, g].double(), v[:, g].double(), dout[:, h].double()
        s = (qh @ kh.t()) * scale
        p = torch.softmax(s, 1)
        o = p @ vh
        # scores in 32 bits, twice (in p and in the sum below it); sums of m terms
        ep = 2 * (size + 4) * u32 * float((qh.abs() @ kh.abs().t()).max()) * scale + (m + 48) * u32
        o_tol = (ep + ut + (m + 4) * u32) * (p @ vh.abs()) + ut * o.abs() + smallest
        dp, delta = do @ vh.t(), (do * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        ds_tol = p * ((size + 4) * u32 * (do.abs() @ vh.abs().t() + (do.abs() * o.abs()).sum(1, keepdim=True)) + (do.abs() * o_tol).sum(1, keepdim=True)) \
            + (ep + ut + 8 * u32) * ds.abs()
        parts = [(0, slice(None), h, scale * (ds @ kh), scale * ((ds_tol + (m + 4) * u32 * ds.abs()) @ kh.abs())),
                 (1, slice(None), g, scale * (ds.t() @ qh), scale * ((ds_tol + (n * heads + 4) * u32 * ds.abs()).t() @ qh.abs())),
                 (2, slice(None), g, p.t() @ do, ((ep + ut + (n * heads + 4) * u32) * p).t() @ do.abs())]
        for i, rows, head, value, tol in parts:
            grads[i][rows, head] += value
            tols[i][rows, head] += tol
    return [(g, t + ut * g.abs()) for g, t in zip(grads, tols)]


@pytest.mark.parametrize("n, m, heads, kv_heads", [(256, 4096, 2, 1), (1024, 1024, 2, 2), (40, 2048, 2, 1), (2048, 300, 3, 1), (7, 5000, 1, 1)])
@pytest.mark.parametrize("power", [0, -7, -10, -13])
def test_small_gradients_in_half_precision(n, m, heads, kv_heads, power):
    """Many keys and a small gradient of the result: p and ds lie under fp16's normal range."""
    from faith_amd import ops
    q, k, v, dout = tensors([n], [m], heads, kv_heads, 64, F16, 21)
    dout = (dout.float() * 2.0 ** power).to(F16)
    packing = ops.Packing([n], [m])
    out, lse = ops.attention(q, k, v, packing, return_lse=True)
    grads = ops.attention_backward(dout, q, k, v, out, lse, packing)
    for name, got, (want, tol) in zip(("dq", "dk", "dv"), grads, small_gradient_reference(q, k, v, dout, 0.125)):
        R.check(name, got, want, tol)
        # and over all of it: three independent roundings (p or ds, delta's, the result's) against one of the result
        once = float((want.to(F16).double() - want).norm())
        assert float((got.double() - want).norm()) <= 3 * once + 1e-5 * float(want.norm()), name


@pytest.mark.parametrize("n, m", [(3, 2), (200, 4), (1, 40)])
def test_large_gradients_in_half_precision(n, m):
    """ds passes fp16's largest value where the gradients do not."""
    from faith_amd import ops
    q, k, v, dout = tensors([n], [m], 2, 1, 64, F16, 22)
    q, k, v = (q.float() / 16).to(F16), (k.float() / 16).to(F16), (v.float() * 4).to(F16)
    dout = (dout.float().clamp(-3.9, 3.9) * 2.0 ** 14).to(F16)
    if n > 100:
        dout[1:] *= 2.0 ** -14          # one row large, the others not: a sum over rows stays in range
    packing = ops.Packing([n], [m])
    out, lse = ops.attention(q, k, v, packing, return_lse=True)
    grads = ops.attention_backward(dout, q, k, v, out, lse, packing)
    r = small_gradient_reference(q, k, v, dout, 0.125)
    p = torch.softmax((q[:, 0].double() @ k[:, 0].double().t()) * 0.125, 1)
    dp = dout[:, 0].double() @ v[:, 0].double().t()
    assert float((p * (dp - (p * dp).sum(1, keepdim=True))).abs().max()) > (65504 if m < 40 else 0)
    for i in (0, 1):
        assert float(r[i][0].abs().max()) < 60000
        R.check("dq dk".split()[i], grads[i], *r[i])


@pytest.mark.parametrize("dtype, size", [(F32, 64), (F32, 128), (BF16, 32), (BF16, 64), (BF16, 96), (BF16, 128), (F16, 80)])
@pytest.mark.parametrize("n, m, heads, kv_heads", [(1, 1, 2, 1), (5, 3, 2, 1), (33, 33, 4, 2), (1, 65, 8, 2), (200, 129, 2, 2), (3, 3000, 2, 1), (700, 700, 8, 8)])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_behind_the_last_sequence_never_come_in(dtype, size, n, m, heads, kv_heads, causal):
    """Neither through a tile's end nor through a load's: all arrays hold NaN behind their last row."""
    from faith_amd import ops
    q, k, v, dout = tensors([n], [m], heads, kv_heads, size, dtype, 31)
    far = lambda t: torch.cat([t, torch.full((200, *t.shape[1:]), math.nan, device="cuda", dtype=dtype)])
    qf, kf, vf, df = (far(t) for t in (q, k, v, dout))
    packing = ops.Packing([n], [m])
    want, lse = ops.attention(q, k, v, packing, causal, return_lse=True)
    got, lse_far = ops.attention(qf, kf, vf, packing, causal, return_lse=True)
    assert torch.equal(got[:n], want) and torch.equal(lse, lse_far) and bool(torch.isfinite(want).all())
    a = ops.attention_backward(dout, q, k, v, want, lse, packing, causal)
    b = ops.attention_backward(df, qf, kf, vf, far(want), lse, packing, causal)
    assert all(torch.equal(x, y[:x.shape[0]]) and bool(torch.isfinite(x).all()) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype, size", [(F32, 64), (BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n", [1, 33, 40, 200])
@pytest.mark.parametrize("causal", [False, True])
def test_a_key_that_no_query_minds(dtype, size, n, causal):
    """A key whose scores are all -infinity has no probability: its gradients are zero, whatever the length of the queries'
    last tile."""
    from faith_amd import ops
    m = n + 3
    q, k, v, dout = tensors([n], [m], 2, 1, size, dtype, 32)
    q[:, :, 0] = -q[:, :, 0].abs() - 0.1
    k[1, :, 0] = math.inf
    packing = ops.Packing([n], [m])
    out, lse = ops.attention(q, k, v, packing, causal, return_lse=True)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    _, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, packing, causal)
    assert bool((dv[1] == 0).all()) and bool((dk[1] == 0).all())
    assert bool(torch.isfinite(dk).all()) and bool(torch.isfinite(dv).all())


def attention_where_seen(q, k, v, lengths, key_lengths, scale, dout):
    """Causal attention and its gradients in float64, every row from what it sees alone: a masked value is never multiplied, not
    even by zero.  A NaN that is seen stays one."""
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = b = 0
    for n, m in zip(lengths, key_lengths):
        for h in range(heads):
            g = h // group
            for i in range(n):
                e = i + m - n + 1
                if e <= 0:
                    continue
                kk, vv, qi, do = k[b:b + e, g], v[b:b + e, g], q[a + i, h], dout[a + i, h]
                p = torch.softmax((kk * qi).sum(1) * scale, 0)
                o = (p[:, None] * vv).sum(0)
                ds = p * ((vv * do).sum(1) - (do * o).sum())
                out[a + i, h] = o
                dq[a + i, h] = scale * (ds[:, None] * kk).sum(0)
                dk[b:b + e, g] += scale * ds[:, None] * qi
                dv[b:b + e, g] += p[:, None] * do
        a, b = a + n, b + m
    return out, dq, dk, dv


@pytest.mark.parametrize("dtype, size", [(F32, 64), (F32, 128), (BF16, 32), (BF16, 64), (BF16, 128), (F16, 64), (F16, 96)])
@pytest.mark.parametrize("lengths, keys, heads, kv_heads", [([50], [50], 2, 1), ([130, 20], [130, 33], 2, 2), ([3], [400], 4, 1), ([40], [25], 2, 1)])
@pytest.mark.parametrize("what", ["k", "v", "q", "dout", "all"])
def test_what_is_no_number_reaches_exactly_those_that_see_it(dtype, size, lengths, keys, heads, kv_heads, what):
    """In the middle of the sequence and in its last place, NaN and infinities: what sees them and what does not lie in one tile."""
    from faith_amd import ops
    q, k, v, dout = tensors(lengths, keys, heads, kv_heads, size, dtype, 51)
    for name, t in (("k", k), ("v", v), ("q", q), ("dout", dout)):
        if what in (name, "all"):
            # a column of its own for each, so that no two infinities meet that the order of a sum could tell apart
            for place, column, bad in ((t.shape[0] // 2, 1, math.nan), (t.shape[0] - 1, 3, math.nan), (t.shape[0] // 3, 2, math.inf)):
                t[place, -1, column] = bad
    packing = ops.Packing(lengths, keys)
    scale = 1 / math.sqrt(size)
    out, lse = ops.attention(q, k, v, packing, causal=True, return_lse=True)
    got = (out, *ops.attention_backward(dout, q, k, v, out, lse, packing, causal=True))
    want = attention_where_seen(q, k, v, lengths, keys, scale, dout)
    clean = [torch.nan_to_num(t, 0, 0, 0) for t in (q, k, v, dout)]
    r = R.attention(*clean[:3], lengths, keys, True, scale, clean[3])
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        finite = torch.isfinite(b)
        assert bool((torch.isfinite(a) == finite).all()), f"{name}: finite at other places than expected"
        # where nothing of it comes in, the error is that of a call without it
        off = torch.where(finite, (a.double() - b).abs() - r[name + "_tol"] * 1.01, 0.0)
        assert bool((off <= 0).all()), f"{name}: off by more than roundings account for"


def test_a_long_prompt_of_what_is_no_number_is_no_slower():
    """A NaN that everything sees, and nothing but NaN (a run that has diverged): the first result stands, and the time is the ordinary one."""
    from faith_amd import ops
    n = 8192
    q, k, v, dout = tensors([n], [n], 8, 2, 64, BF16, 52)
    packing = ops.Packing([n])

    def run(*t):
        out, lse = ops.attention(*t[:3], packing, causal=True, return_lse=True)
        return (out, *ops.attention_backward(t[3], *t[:3], out, lse, packing, causal=True))

    def milliseconds(*t):
        run(*t)
        times = []
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            got = run(*t)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times), got
    usual, _ = milliseconds(q, k, v, dout)
    k[0], v[0] = math.nan, math.nan
    took, got = milliseconds(q, k, v, dout)
    assert all(bool(torch.isnan(t[1:]).all()) for t in got) and took <= 2 * usual
    nothing = [torch.full_like(t, math.nan) for t in (q, k, v, dout)]
    took, got = milliseconds(*nothing)
    assert all(bool(torch.isnan(t[1:]).all()) for t in got) and took <= 2 * usual


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, m, causal", [(3, 1, False), (1, 1, True), (200, 1, False), (40, 40, True)])
def test_a_score_that_is_no_number_has_no_gradient_that_is_one(dtype, n, m, causal):
    """One key alone: dq = 0 because its probability is 1, which it is not where the score is NaN or infinite."""
    from faith_amd import ops
    for bad in (math.nan, math.inf, -math.inf):
        q, k, v, dout = tensors([n], [m], 1, 1, 64, dtype, 41)
        q[0, 0, 3] = bad
        packing = ops.Packing([n], [m])
        out, lse = ops.attention(q, k, v, packing, causal, return_lse=True)
        dq, dk, _ = ops.attention_backward(dout, q, k, v, out, lse, packing, causal)
        assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(dq[0]).all()) and bool(torch.isnan(dk[0]).any())
        alone = dq[1:] if m == 1 else dq[:0]
        assert bool((alone == 0).all()) and bool(torch.isfinite(out[1:]).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, m, heads, causal", [(5, 7, 2, False), (200, 300, 2, True), (1, 9000, 1, False), (128, 9000, 1, True), (700, 64, 4, False)])
def test_scores_that_are_all_minus_infinity_give_no_number(dtype, n, m, heads, causal):
    """softmax of nothing but -infinity is 0 / 0; only a row that sees no key at all is zero."""
    from faith_amd import ops
    q, k, v, dout = tensors([n], [m], heads, 1, 64, dtype, 42)
    q[:, :, 0], k[:, :, 0] = 1, -math.inf
    q[0, :, 0] = -1                                             # all +infinity: as little a number
    packing = ops.Packing([n], [m])
    out, lse = ops.attention(q, k, v, packing, causal, return_lse=True)
    assert bool(torch.isnan(out).all()) and bool((lse[:, 1:] == -math.inf).all())
    grads = ops.attention_backward(dout, q, k, v, out, lse, packing, causal)
    assert bool(torch.isnan(grads[0]).all()) and bool(torch.isnan(grads[2]).all())
    # beside rows that see none, and a sequence of ordinary ones
    packing = ops.Packing([n, 9, 6], [m, 4, 6])
    q, k, v, dout = (torch.cat([a, b]) for a, b in zip((q, k, v, dout), tensors([9, 6], [4, 6], heads, 1, 64, dtype, 43)))
    out, lse = ops.attention(q, k, v, packing, True, return_lse=True)
    assert bool(torch.isnan(out[:n]).all()) == (n <= m) and bool((out[n:n + 5] == 0).all()) and bool(torch.isfinite(out[n:]).all())
    assert bool((lse[:, n:n + 5] == -math.inf).all())


def test_one_token_into_a_result_of_any_strides():
    from faith_amd import ops
    q, k, v, _ = tensors([1], [9], 4, 2, 32, BF16, 61)
    packing = ops.Packing([1], [9])
    want = ops.attention(q, k, v, packing)
    store = torch.zeros(1 << 20, device="cuda", dtype=BF16)
    for rows, strides in ((1, (8, 32, 1)), (1, (160, 40, 1)), (16, (40, 32, 1)), (16, (32, 1 << 14, 1)), (1, (1 << 10, 1 << 18, 1))):
        out = store.as_strided((rows, 4, 32), strides)
        assert torch.equal(ops.attention(q, k, v, packing, out=out)[:1], want)
