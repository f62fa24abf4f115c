"""The residual norm of the concrete pass against its definition in float64 (tests/concrete_reference.py)."""
import math

import pytest
import torch

from tests import concrete_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROWS = [(1, 8), (3, 7), (5, 64), (960, 256), (17, 512), (9, 1000), (33, 1032), (4, 2048), (7, 4096), (5, 5120), (3, 8200), (2, 16384), (2, 20000), (1000, 78), (1, 1)]


def tensors(rows, n, dtype, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, residual, dy, dsum = (rnd(rows, n).to(dtype) for _ in range(4))
    return x, residual, (1 + 0.1 * rnd(n)).to(dtype), (0.1 * rnd(n)).to(dtype) if bias else None, dy, dsum


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["rms", "standard", "no_var"])
@pytest.mark.parametrize("rows, n", ROWS)
def test_norm_and_gradients(rows, n, kind, dtype):
    from faith_amd import ops
    x, residual, w, b, dy, dsum = tensors(rows, n, dtype, rows + n)
    y, h, stats = ops.residual_norm(x, residual, w, b, kind, 1e-6, return_stats=True)
    r = R.norm(x, residual, w, b, kind, 1e-6, dy, dsum)
    R.check("y", y, r["y"], r["y_tol"])
    R.check("h", h, r["h"], r["h_tol"])
    dx, dw, db = ops.residual_norm_backward(dy, h, w, stats, kind, dsum, with_bias=True)
    for name, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
        R.check(name, got, r[name], r[name + "_tol"])
    again = ops.residual_norm_backward(dy, h, w, stats, kind, dsum, with_bias=True)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]) and torch.equal(db, again[2])
    # one gradient less is the same others
    only = ops.residual_norm_backward(dy, h, w, stats, kind, dsum, with_weight=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None
    only = ops.residual_norm_backward(dy, h, w, stats, kind, dsum, with_weight=False, with_bias=True)
    assert only[1] is None and torch.equal(only[2], db)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, n", [(5, 256), (3, 1111), (4, 4096)])
def test_every_operand_may_be_left_out(rows, n, dtype):
    from faith_amd import ops
    x, residual, w, b, dy, dsum = tensors(rows, n, dtype, 4)
    for res in (None, residual):
        for weight in (None, w):
            for bias in (None, b):
                y, h, stats = ops.residual_norm(x, res, weight, bias, "standard", 1e-6, return_stats=True)
                r = R.norm(x, res, weight, bias, "standard", 1e-6, dy)
                R.check("y", y, r["y"], r["y_tol"])
                assert res is not None or h is x
                dx, dw, _ = ops.residual_norm_backward(dy, h, weight, stats, "standard", with_weight=weight is not None)
                R.check("dx", dx, r["dx"], r["dx_tol"])
                if weight is not None:
                    R.check("dweight", dw, r["dweight"], r["dweight_tol"])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bits", ["int8", "e4m3"])
@pytest.mark.parametrize("rows, n", [(5, 64), (3, 7), (33, 1032), (7, 4096), (2, 20000)])
def test_eight_bits(rows, n, bits, dtype):
    """A value is within half a step of what it stands for (int8: the scale; e4m3: 2^-4 of the value, 2^-10 steps under the
    normal range), beyond what y itself is off by; the largest of a row is the end of the range."""
    from faith_amd import ops
    x, residual, w, b, _, _ = tensors(rows, n, dtype, 11)
    x[0], residual[0] = 0, 0
    if b is not None:
        b = torch.zeros_like(b) if rows > 3 else b
    q, scales, h = ops.residual_norm(x, residual, w, b, "rms", 1e-6, quantize=bits)
    assert q.dtype == (torch.int8 if bits == "int8" else torch.float8_e4m3fn) and scales.shape == (rows,) and q.shape == x.shape
    r = R.norm(x, residual, w, b, "rms", 1e-6)
    top = r["y"].abs().amax(1)
    most = 127.0 if bits == "int8" else 448.0
    R.check("scale", scales, top / most, r["y_exact_tol"].amax(1) / most + 2 * R.U32 * top / most + 1e-30)
    assert torch.equal(h, ops.residual_norm(x, residual, w, b, "rms", 1e-6)[1])
    s = scales.double()[:, None]
    half = s / 2 if bits == "int8" else torch.maximum(r["y"].abs() * 2.0 ** -4, s * 2.0 ** -10)
    R.check("values", q.float().double() * s, r["y"], half * (1 + 1e-5) + r["y_exact_tol"] + 1e-30)
    full = q.float().abs().amax(1)
    assert bool((full[top > 0] == most).all())
    if rows > 3:
        assert float(scales[0]) == 0 and bool((q[0].float() == 0).all())


def test_eight_bits_of_values_that_lie_on_the_steps():
    """y = q exactly: root mean square of a row of +-1 is 1, so y is the weight."""
    from faith_amd import ops
    w = torch.arange(-127, 129, device="cuda", dtype=torch.float32).clamp_max(127)
    x = torch.ones(2, 256, device="cuda")
    q, scales, _ = ops.residual_norm(x, None, w, None, "rms", 0.0, quantize="int8")
    assert bool((scales == 1).all()) and torch.equal(q[0].float(), w)
    # halves go to the even neighbour
    w = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 3.5], device="cuda")
    q, _, _ = ops.residual_norm(torch.ones(1, 8, device="cuda"), None, w, None, "rms", 0.0, quantize="int8")
    assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -2, 4]
    w = torch.tensor([448.0, 17.0, 19.0, 21.0, -17.0, 0.001953125, 0.0009765625, 0.0029296875], device="cuda")
    q, _, _ = ops.residual_norm(torch.ones(1, 8, device="cuda"), None, w, None, "rms", 0.0, quantize="e4m3")
    assert torch.equal(q[0].float(), w.to(torch.float8_e4m3fn).float())


def test_rows_that_hold_no_numbers():
    from faith_amd import ops
    x = torch.randn(4, 64, device="cuda")
    x[1, 3], x[2, 5] = math.nan, math.inf
    y, _ = ops.residual_norm(x, None, None, None, "rms")
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[3]).all())
    for bits in ("int8", "e4m3"):
        q, s, _ = ops.residual_norm(x, None, None, None, "rms", quantize=bits)
        a, b = ops.residual_norm(x[::3].contiguous(), None, None, None, "rms", quantize=bits)[:2]
        assert torch.equal(q[::3].float(), a.float()) and torch.equal(s[::3], b)


def test_a_large_mean_does_not_cancel_the_variance():
    from faith_amd import ops
    x = torch.randn(8, 768, device="cuda") + 1000
    r = R.norm(x, None, None, None, "standard", 1e-12)
    y, _ = ops.residual_norm(x, None, None, None, "standard", 1e-12)
    # the mean is known to some 768 half steps of 1000 at worst, which moves z; the variance stays that of the centred values
    R.check("y", y, r["y"], r["y_tol"])


@pytest.mark.parametrize("offset", [0, 1])
def test_rows_off_the_16_byte_grid(offset):
    from faith_amd import ops
    rows, n = 6, 512
    make = lambda: torch.randn(rows * n + 8, device="cuda").to(BF16)[offset:offset + rows * n].view(rows, n)
    x, residual, dy = make(), make(), make()
    w = torch.randn(n + 8, device="cuda").to(BF16)[offset:offset + n]
    y, h, stats = ops.residual_norm(x, residual, w, None, "rms", 1e-6, return_stats=True)
    r = R.norm(x, residual, w, None, "rms", 1e-6, dy)
    R.check("y", y, r["y"], r["y_tol"])
    dx, dw, _ = ops.residual_norm_backward(dy, h, w, stats, "rms")
    R.check("dx", dx, r["dx"], r["dx_tol"])
    R.check("dweight", dw, r["dweight"], r["dweight_tol"])


def test_gradients_against_differences():
    """Central differences of the definition in float64 along random directions."""
    from faith_amd import ops
    x, residual, w, b, dy, dsum = tensors(7, 96, F32, 3)
    for kind in ("rms", "standard", "no_var"):
        y, h, stats = ops.residual_norm(x, residual, w, b, kind, 1e-6, return_stats=True)
        dx, dw, db = ops.residual_norm_backward(dy, h, w, stats, kind, dsum, with_bias=True)

        def loss(x, w, b):
            r = R.norm(x, residual.double(), w, b, kind, 1e-6)
            return float((r["y"] * dy.double()).sum() + (r["h"] * dsum.double()).sum())
        base, step = [t.double() for t in (x, w, b)], 1e-4
        g = torch.Generator(device="cuda").manual_seed(7)
        for i, grad in enumerate((dx, dw, db)):
            d = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
            d /= d.norm()
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + step * d, base[i] - step * d
            want = (loss(*up) - loss(*down)) / (2 * step)
            assert abs(float((grad.double() * d).sum()) - want) <= 1e-5 * float(grad.norm()) + 1e-6


def test_no_rows():
    from faith_amd import ops
    x = torch.zeros(0, 64, device="cuda", dtype=BF16)
    w = torch.ones(64, device="cuda", dtype=BF16)
    y, h, stats = ops.residual_norm(x, x, w, None, "rms", return_stats=True)
    dx, dw, _ = ops.residual_norm_backward(x, h, w, stats, "rms")
    assert y.shape == (0, 64) and dx.shape == (0, 64) and bool((dw == 0).all())


def test_captured_and_replayed_between_eager_work():
    from faith_amd import ops
    x, residual, w, b, dy, dsum = tensors(300, 1024, BF16, 3)

    def body():
        y, h, stats = ops.residual_norm(x, residual, w, b, "standard", 1e-6, return_stats=True)
        return (y, h, *ops.residual_norm_backward(dy, h, w, stats, "standard", dsum, with_bias=True),
                *ops.residual_norm(x, residual, w, b, "rms", 1e-6, quantize="e4m3"))
    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = body()
    for _ in range(4):
        x.copy_(torch.randn(x.shape, device="cuda").to(BF16))
        want = body()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.float(), b_.float()) for a, b_ in zip(want, result))


def test_leading_axes_and_refusals():
    from faith_amd import ops
    x, residual, w, b, dy, _ = tensors(12, 64, F32, 3)
    shaped = ops.residual_norm(x.view(3, 4, 64), residual.view(3, 4, 64), w, b, "standard", return_stats=True)
    flat = ops.residual_norm(x, residual, w, b, "standard", return_stats=True)
    assert torch.equal(shaped[0].view(12, 64), flat[0]) and shaped[2].shape == (3, 4)
    for args, kw, kind, what in [((x, residual[:3]), {}, ValueError, "residual"), ((x, residual.half()), {}, TypeError, "residual"), ((x, None, w[:5]), {}, ValueError, "weight"),
                                 ((x.t(),), {}, ValueError, "contiguous"), ((x.double(),), {}, TypeError, "x:"), ((x,), dict(kind="batch"), ValueError, "kind"),
                                 ((x,), dict(quantize="int4"), ValueError, "quantize"), ((x,), dict(eps=-1e-6), ValueError, "eps"), ((x,), dict(eps=math.nan), ValueError, "eps")]:
        with pytest.raises(kind, match=what):
            ops.residual_norm(*args, **kw)
    with pytest.raises(ValueError, match="stats"):
        ops.residual_norm_backward(dy, x, w, flat[2][:3], "standard")
    with pytest.raises(ValueError, match="dy"):
        ops.residual_norm_backward(dy[:3], x, w, flat[2], "standard")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bits", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["rms", "standard", "no_var"])
@pytest.mark.parametrize("n", [64, 63, 1032, 4096, 8200, 20000])
def test_eight_bits_of_rows_that_hold_no_numbers(n, kind, bits, dtype):
    """A row with a NaN, or with an infinity, stands for no number anywhere: no finite scale, NaN in e4m3, and NaN whichever way it
    is read back.  On the way that keeps the row in registers and on that for any width."""
    from faith_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(6, n, generator=g, device="cuda").to(dtype)
    clean = ops.residual_norm(x, None, None, None, kind, quantize=bits)
    x[1, 3], x[2, n - 1], x[4, 5] = math.nan, math.inf, -math.inf
    q, scales, _ = ops.residual_norm(x, None, None, None, kind, quantize=bits)
    for row in (1, 2, 4):
        assert bool(torch.isnan(scales[row])) and bool(torch.isnan(q[row].float() * scales[row]).all())
        assert bool((q[row].float() == 0).all()) if bits == "int8" else bool(torch.isnan(q[row].float()).all())
    for row in (0, 3, 5):
        assert torch.equal(q[row].float(), clean[0][row].float()) and torch.equal(scales[row], clean[1][row])
    # an infinite weight: an infinity, and none of the row's numbers has a finite scale
    w = torch.ones(n, device="cuda", dtype=dtype)
    w[7] = math.inf
    q, scales, _ = ops.residual_norm(x[:1], None, w, None, kind, quantize=bits)
    assert not bool(torch.isfinite(scales).any()) and bool(torch.isnan(q.float() * scales[:, None]).all())


@pytest.mark.parametrize("n", [(1 << 31) + 8, (1 << 32) + 64])
def test_rows_longer_than_32_bits_count_are_refused(n):
    """Not taken for the shorter row that their length is in 32 bits."""
    from faith_amd import ops
    x = torch.empty(1, n, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.residual_norm(x)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.residual_norm_backward(x, x, None, torch.ones(1, device="cuda"), with_weight=False)
