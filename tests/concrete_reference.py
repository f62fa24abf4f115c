"""Plain float64 implementations of the concrete pass's operators, and how far a kernel may be off.

The tolerances count roundings.  u is half a step of a type relative to the value (torch.finfo(t).eps / 2): u32 for sums and
softmax values, ut for what is rounded to the operands' type.  A sum of n terms in 32 bits, in any order, is off by at most
n u32 times the sum of the terms' magnitudes.
"""
import math

import torch

U32 = torch.finfo(torch.float32).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, lengths, key_lengths, causal, scale, dout=None):
    """Packed attention in float64 on the operands' device, head by head.  Returns a dict with out, lse and, with dout, dq, dk,
    dv, each with its elementwise tolerance under the name + "_tol"."""
    dtype = q.dtype
    ut = half_step(dtype)
    two_bytes = dtype != torch.float32
    # what a value under the type's normal range may be off by, beyond ut of itself
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q64, k64, v64 = q.double(), k.double(), v.double()
    heads, group, size = q.shape[1], q.shape[1] // k.shape[1], q.shape[2]
    r = {n: torch.zeros_like(t) for n, t in (("out", q64), ("dq", q64), ("dk", k64), ("dv", v64))}
    r.update({n + "_tol": torch.zeros_like(t) for n, t in list(r.items())})
    r["lse"] = torch.full((heads, sum(lengths)), -math.inf, dtype=torch.float64, device=q.device)
    r["lse_tol"] = torch.zeros_like(r["lse"])
    a = b = 0
    for n, m in zip(lengths, key_lengths):
        if n and m:
            place = torch.arange(n, device=q.device)[:, None] + (m - n)
            allowed = torch.arange(m, device=q.device)[None, :] <= (place if causal else m)
            for h in range(heads):
                g = h // group
                qh, kh, vh = q64[a:a + n, h], k64[b:b + m, g], v64[b:b + m, g]
                s = torch.where(allowed, (qh @ kh.t()) * scale, -math.inf)
                top = s.amax(1, keepdim=True)
                e = torch.where(allowed, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
                total = e.sum(1, keepdim=True)
                p = e / torch.where(total == 0, 1.0, total)
                mag, o = p @ vh.abs(), p @ vh
                r["out"][a:a + n, h] = o
                some = total[:, 0] > 0
                r["lse"][h, a:a + n] = torch.where(some, top[:, 0] + torch.log(torch.where(some, total[:, 0], 1.0)), -math.inf)
                # a score: `size` products and sums, its scaling and the difference to the reference
                sabs = (qh.abs() @ kh.abs().t()) * scale
                es = (size + 4) * U32 * torch.where(allowed, sabs, 0.0).amax(1, keepdim=True)
                # a probability: the score's error above and in the sum below, the exponential, the sum of m terms
                ep = 2 * es + (m + 16) * U32
                rounded = ut if two_bytes else 0.0
                out_tol = (ep + rounded + (m + 4) * U32) * mag + tiny * vh.abs().sum(0) + ut * o.abs() + tiny
                r["out_tol"][a:a + n, h] = out_tol
                r["lse_tol"][h, a:a + n] = (es + (m + 16) * U32)[:, 0] + 4 * U32 * torch.nan_to_num(r["lse"][h, a:a + n], 0, 0, 0).abs()
                if dout is None:
                    continue
                do = dout[a:a + n, h].double()
                dp = do @ vh.t()
                delta = (do * o).sum(1, keepdim=True)
                ds = p * (dp - delta)
                # delta comes from the stored result, which is off by its tolerance
                dp_tol = (size + 4) * U32 * (do.abs() @ vh.abs().t())
                delta_tol = (size + 4) * U32 * (do.abs() * o.abs()).sum(1, keepdim=True) + (do.abs() * out_tol).sum(1, keepdim=True)
                lse_err = 2 * es + (m + 32) * U32
                ds_tol = p * (dp_tol + delta_tol) + (lse_err + 4 * U32 + rounded) * ds.abs() + tiny
                p_tol = (lse_err + rounded) * p + tiny
                r["dq"][a:a + n, h] = scale * (ds @ kh)
                r["dq_tol"][a:a + n, h] = scale * ((ds_tol + (m + 4) * U32 * ds.abs()) @ kh.abs())
                terms = n * group
                r["dk"][b:b + m, g] += scale * (ds.t() @ qh)
                r["dk_tol"][b:b + m, g] += scale * ((ds_tol + (terms + 4) * U32 * ds.abs()).t() @ qh.abs())
                r["dv"][b:b + m, g] += p.t() @ do
                r["dv_tol"][b:b + m, g] += (p_tol + (terms + 4) * U32 * p).t() @ do.abs()
        a, b = a + n, b + m
    if dout is not None:
        for name in ("dq", "dk", "dv"):
            r[name + "_tol"] += ut * r[name].abs() + tiny + 1e-30
    r["out_tol"] += 1e-30
    return r


def check(name, got, want, tol):
    got = got.double()
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)}, expected {tuple(want.shape)}"
    finite = torch.isfinite(want)
    assert bool((torch.isfinite(got) == finite).all()), f"{name}: finite at other places than expected"
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), f"{name}: NaN at other places than expected"
    off = torch.where(finite, (got - want).abs() / tol, 0.0)
    assert bool((off <= 1).all()), f"{name}: off by {float(off.max()):.3g} times what roundings account for"


def norm(x, residual, weight, bias, kind, eps, dy=None, dsum=None):
    """The residual norm in float64 with tolerances, as above; x [rows, n]."""
    n, ut, dtype = x.shape[-1], half_step(x.dtype), x.dtype
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    h = x.double() + (residual.double() if residual is not None else 0.0)
    w = weight.double() if weight is not None else torch.ones(n, dtype=torch.float64, device=x.device)
    b = bias.double() if bias is not None else torch.zeros(n, dtype=torch.float64, device=x.device)
    mean = h.mean(-1, keepdim=True) if kind != "rms" else torch.zeros_like(h[..., :1])
    c = h - mean
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt() if kind != "no_var" else torch.ones_like(mean)
    z = c * rstd
    y = z * w + b
    # h is one rounding, the mean a sum of n; the centred values inherit both, the variance twice that relative to itself
    c_tol = U32 * (h.abs() + c.abs()) + (n + 2) * U32 * h.abs().mean(-1, keepdim=True) * (kind != "rms")
    spread = c.square().mean(-1, keepdim=True) + eps
    rstd_rel = ((n + 4) * U32 + (c.abs() * c_tol).mean(-1, keepdim=True) / spread) if kind != "no_var" else torch.zeros_like(mean)
    z_tol = c_tol * rstd + z.abs() * (rstd_rel + 4 * U32)
    y_tol = z_tol * w.abs() + 4 * U32 * ((z * w).abs() + b.abs())
    r = dict(h=h, h_tol=ut * h.abs() + U32 * h.abs() + tiny, y=y, y_exact_tol=y_tol, y_tol=y_tol + ut * y.abs() + tiny, z=z, rstd=rstd)
    if dy is None:
        return r
    # the gradient takes h as it was stored: rounded to the type where there was a residual
    stored = (ut if residual is not None else 0.0) * h.abs() * rstd
    z_tol = z_tol + stored
    dy = dy.double()
    g = dy * w
    m0 = g.mean(-1, keepdim=True) if kind != "rms" else torch.zeros_like(mean)
    m1 = (g * z).mean(-1, keepdim=True) if kind != "no_var" else torch.zeros_like(mean)
    dh = (g - m0 - z * m1) * rstd
    m0_tol = (n + 2) * U32 * g.abs().mean(-1, keepdim=True) * (kind != "rms")
    m1_tol = ((n + 4) * U32 * (g * z).abs().mean(-1, keepdim=True) + (g.abs() * z_tol).mean(-1, keepdim=True)) * (kind != "no_var")
    dh_tol = (4 * U32 * (g.abs() + m0.abs() + (z * m1).abs()) + m0_tol + z.abs() * m1_tol + z_tol * m1.abs()) * rstd + dh.abs() * (rstd_rel + 2 * U32)
    dx = dh + (dsum.double() if dsum is not None else 0.0)
    rows = max(1, x.numel() // n)
    flat = lambda t: t.reshape(-1, n)
    dw, db = flat(dy * z).sum(0), flat(dy).sum(0)
    r.update(dx=dx, dx_tol=dh_tol + 2 * U32 * dx.abs() + ut * dx.abs() + tiny,
             dweight=dw, dweight_tol=flat(dy.abs() * z_tol).sum(0) + (rows + 2) * U32 * flat((dy * z).abs()).sum(0) + ut * dw.abs() + tiny,
             dbias=db, dbias_tol=(rows + 2) * U32 * flat(dy.abs()).sum(0) + ut * db.abs() + tiny)
    return r
