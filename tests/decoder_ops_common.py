"""Float64 forms of the decoder operators with, for every output, a bound on what the kernels may be
off by: what each of their roundings can change, carried through absolute values.

u is half a step of the element type (torch.finfo(t).eps / 2), f = 2^-24 that of float32."""
import math

import torch

F = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the smallest numbers of the type: a rounding is off by at most this
    where the relative bound ends."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got = got.double()
    assert bool(torch.isfinite(got).all()), "%s: not finite" % name
    bad = (got - want).abs() - bound
    assert bool((bad <= 0).all()), "%s: off by %g where %g is allowed (%d of %d elements)" % (
        name, float((got - want).abs().flatten()[bad.argmax()]),
        float(bound.expand_as(want).flatten()[bad.argmax()]), int((bad > 0).sum()), bad.numel())


# ---------------------------------------------------------------------------------- layer norm
def layer_norm(x, weight, bias, residual, eps, dy=None):
    """[(name, value, bound)].  A row's sum is a chain of at most 32 additions per thread and a
    tree of ten: the mean is off by h f mean|s| with h = 48, the deviations by that and a rounding,
    the standard deviation relatively by what its deviations are plus h f."""
    u, h = half_step(x.dtype), 48
    s = x.double() + (0 if residual is None else residual.double())
    n = s.shape[-1]
    w = torch.ones(n, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    mean = s.mean(-1, keepdim=True)
    var = ((s - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (s - mean) * rstd
    e_dev = F * (h * s.abs().mean(-1, keepdim=True) + 2 * s.abs())      # s - mean
    # d rstd / rstd = -mean(c dc) rstd^2, |.| <= sqrt(mean dc^2) rstd
    e_rstd = (e_dev ** 2).mean(-1, keepdim=True).sqrt() * rstd + (h + 8) * F
    e_xh = e_dev * rstd + xh.abs() * e_rstd + 2 * F * xh.abs()
    y = xh * w + b
    out = [("y", y, u * y.abs() + 2 * F * (xh * w).abs() + e_xh * w.abs() + tiny(x.dtype))]
    if dy is None:
        return out
    g = dy.double()
    t = g * w
    m0, m1 = t.mean(-1, keepdim=True), (t * xh).mean(-1, keepdim=True)
    dx = rstd * (t - m0 - xh * m1)
    size = t.abs() + t.abs().mean(-1, keepdim=True) + xh.abs() * (t * xh).abs().mean(-1, keepdim=True)
    e_m1 = (t.abs() * e_xh).mean(-1, keepdim=True)
    e = rstd * ((h + 8) * F * size + e_xh * m1.abs() + xh.abs() * e_m1) + dx.abs() * e_rstd
    out.append(("dx", dx, u * dx.abs() + 1.01 * e + tiny(x.dtype)))
    rows = lambda v: v.reshape(-1, n)
    # the column sums: a chain of rows per thread (at most rows / 64 + 8), then of partial rows
    chain = (rows(g).shape[0] / 64 + 8 + 160) * F
    dw, db = rows(g * xh).sum(0), rows(g).sum(0)
    out.append(("dw", dw, u * dw.abs() + rows(g.abs() * e_xh).sum(0) + chain * rows((g * xh).abs()).sum(0)
                + tiny(x.dtype)))
    out.append(("db", db, u * db.abs() + chain * rows(g.abs()).sum(0) + tiny(x.dtype)))
    return out


# ------------------------------------------------------------------------------------- linear
def _sum_bound(length, f32):
    """Relative to the sum of absolute products: the matrix instructions add 16 products at a time
    (six times as many for split float32, which also drops three terms of 2^-24), shares of the
    sum are added last."""
    return (length / 16 * (6 if f32 else 1) + 40) * F + (4 * F if f32 else 0)


def linear(x, weight, bias, act, residual, dy=None):
    dtype = x.dtype
    u, f32 = half_step(dtype), dtype == torch.float32
    X, W = x.double().reshape(-1, x.shape[-1]), weight.double()
    n, k = W.shape
    m = X.shape[0]
    z = X @ W.t()
    ez = _sum_bound(k, f32) * (X.abs() @ W.abs().t())
    if bias is not None:
        z = z + bias.double()
        ez = ez + F * z.abs()
    cdf = torch.special.erfc(-z / math.sqrt(2)) / 2
    pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "relu":
        a, slope, ea = z.clamp(min=0), (z > 0).double(), ez
    elif act == "gelu":    # |gelu'| <= 1.13; the kernel's tail Phi(-|z|): 40 f relative, for 16-bit types
        # 2^-14 (the fit's 4e-5, and f z^2 for the exponential's argument); gelu = max(z, 0) - |z| Phi(-|z|)
        a, slope = z * cdf, cdf + z * pdf
        tail = torch.special.erfc(z.abs() / math.sqrt(2)) / 2
        ea = 1.13 * ez + (40 * F if f32 else 2.0 ** -14 + z * z * F) * z.abs() * tail + 2 * F * a.abs()
    else:
        a, slope, ea = z, torch.ones_like(z), ez
    y = a if residual is None else a + residual.double().reshape(m, n)
    shape = x.shape[:-1] + (n,)
    out = [("y", y.reshape(shape), ((u + F) * y.abs() + ea + tiny(dtype)).reshape(shape))]
    if dy is None:
        return out
    g = dy.double().reshape(m, n)
    dz = g * slope
    if act == "relu":      # z within its error of zero may fall on either side
        edz = g.abs() * (z.abs() <= ez + tiny(dtype)).double()
    elif act == "gelu":    # |gelu''| <= 0.8; the slope's own arithmetic 2^-20, and its rounding, f32's
        # half step (16 bits: the tail, at most a half, to 2^-14, and half a fixed-point step, 2^-16)
        own = 2.0 ** -20 + F * slope.abs() if f32 else 2.0 ** -15 + 2.0 ** -16
        edz = g.abs() * (0.8 * ez + own) + u * dz.abs() + tiny(dtype)
    else:
        edz = torch.zeros_like(g)
    dx, dw, db = dz @ W, dz.t() @ X, dz.sum(0)
    # (a bound of dz is a bound of what enters the sums' own roundings as well: the factor 1.01)
    big = 1.01 * dz.abs() + edz
    out.append(("dx", dx.reshape(x.shape), (u * dx.abs() + edz @ W.abs() + _sum_bound(n, f32) * (
        big @ W.abs()) + tiny(dtype)).reshape(x.shape)))
    out.append(("dw", dw, u * dw.abs() + edz.t() @ X.abs() + _sum_bound(m, f32) * (big.t() @ X.abs())
                + tiny(dtype)))
    if bias is not None:
        chain = (m / 32 + 80) * F
        out.append(("db", db, u * db.abs() + edz.sum(0) + chain * big.sum(0) + tiny(dtype)))
    if residual is not None:
        out.append(("dres", g.reshape(shape), torch.zeros_like(g).reshape(shape)))
    return out


# ---------------------------------------------------------------------------- cross-attention
def live_keys(k, lengths, mask):
    """(B, Lk) bool"""
    B, Lk = k.shape[:2]
    live = torch.ones((B, Lk), dtype=torch.bool, device=k.device)
    if lengths is not None:
        live &= torch.arange(Lk, device=k.device)[None] < lengths[:, None]
    if mask is not None:
        live &= ~mask
    return live


def cross_attention(q, k, v, lengths, mask, scale, dy=None):
    dtype = q.dtype
    u = 0.0 if dtype == torch.float32 else half_step(dtype)      # of P and dS inside
    uo = half_step(dtype)
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    live = live_keys(k, lengths, mask)[:, None, None, :]
    dead = ~live_keys(k, lengths, mask)[:, :, None, None]
    Q = q.double().permute(0, 2, 1, 3)                            # (B, H, Lq, D)
    K, V = (t.double().masked_fill(dead, 0.0).repeat_interleave(G, 2).permute(0, 2, 1, 3)
            for t in (k, v))
    s = scale * (Q @ K.transpose(-1, -2))
    s = s.masked_fill(~live, float("-inf"))
    top = s.amax(-1, keepdim=True) if Lk else s.sum(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot > 0, tot, torch.ones_like(tot))
    out = p @ V
    # a score: D products in f32, its scaling, the subtraction of the maximum and the exponential's
    # argument; relative error of P from both the row's own score and the sum's
    size = (scale * (Q.abs() @ K.abs().transpose(-1, -2))).amax(-1, keepdim=True) if Lk else tot
    ep = 2 * ((D / 2 + 8) * F * size + (Lk / 16 + 40) * F)
    # ... and absolutely: the exponential instruction returns 0 for results below 2^-126, and P <= 1
    # is e^(s - max) (forward) or e^(s - max) / sum (backward) with 1 <= sum, so what is lost of a P is
    # below 2^-126; a 16-bit P loses half the type's smallest step instead (backward, float16: of
    # 2^15 P)
    half = dtype == torch.float16
    ea = max(2.0 ** -126, tiny(dtype) if u else 0.0) * (p > 0).double()
    ea_back = ea * 2.0 ** -15 if half else ea
    back = lambda t: t.permute(0, 2, 1, 3)
    eo = (ep + u) * (p @ V.abs()) + uo * out.abs() + tiny(dtype) + ea @ V.abs()
    res = [("out", back(out), back(eo))]
    if dy is None:
        return res
    g = dy.double().permute(0, 2, 1, 3)
    dp = g @ V.transpose(-1, -2)
    delta = (g * out).sum(-1, keepdim=True)
    e_dp = (D / 2 + 8) * F * (g.abs() @ V.abs().transpose(-1, -2))
    e_delta = (g.abs() * eo).sum(-1, keepdim=True) + D * F * (g.abs() * out.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # (dS itself is rounded once more, in steps of its own that end at 2^-126 or the type's half step;
    # float16: of dS times 2^(5 - e) for dq, 2^(9 - e' - f) for dk, where 2^e, 2^e' and 2^f are above
    # the row's, all rows' and the key's largest |dout|, |dout| and |v|: |x| < 2^e <= 2 |x|)
    e_ds = p * (ep * (dp - delta).abs() + e_dp + e_delta) + (u + 2 * F) * ds.abs() + \
        2.0 ** -126 * (p > 0) * (dp - delta).abs()
    ea_q = ea_k = ea
    if half:
        most, vmost = g.abs().amax(-1, keepdim=True), V.abs().amax(-1)[:, :, None]
        none = lambda t: torch.where(t > 0, 2 * t, torch.ones_like(t))        # (0: 2^0)
        ea_q = ea * none(most) * 2.0 ** -5
        ea_k = ea * none(most.reshape(B, -1).amax(-1)[:, None, None, None]) * none(vmost) * 2.0 ** -9
    fold = lambda t: t.reshape(B, Hk, G, Lk, D).sum(2).permute(0, 2, 1, 3)
    acc = lambda length: (length / 2 + 40) * F                    # the sums of the last products
    dq = scale * (ds @ K)
    e_dq = scale * ((e_ds + ea_q + acc(Lk) * ds.abs()) @ K.abs()) + uo * dq.abs() + tiny(dtype)
    st, et = ds.transpose(-1, -2), (e_ds + ea_k).transpose(-1, -2)
    dk = fold(scale * (st @ Q))
    e_dk = fold(scale * ((et + acc(Lq * G) * st.abs()) @ Q.abs())) + uo * dk.abs() + tiny(dtype)
    pt = p.transpose(-1, -2)
    dv = fold(pt @ g)
    e_dv = fold(((u + ep.transpose(-1, -2) + acc(Lq * G)) * pt + ea_back.transpose(-1, -2)) @ g.abs())
    e_dv = e_dv + uo * dv.abs() + tiny(dtype)
    return res + [("dq", back(dq), back(e_dq)), ("dk", dk, e_dk), ("dv", dv, e_dv)]
