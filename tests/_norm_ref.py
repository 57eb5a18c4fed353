"""Group norm with its activation in float64 from its formulas (test infrastructure).

``reference`` returns every output of the forward, the backward and the double backward as a pair
(value, magnitude).  The magnitude is what the value becomes when no term cancels: every product
and sum taken over absolute values.  An evaluation in fp32 that rounds relative to its own terms
``n`` times in a row is off by at most about n * 2^-24 * magnitude.

``bound`` is that with n = 256 -- at most 128 values of a channel are added one after another by a
thread, some 20 additions fold threads and chunks (the chunks in float64), and the elementwise pass
and its coefficients round fewer than 60 times -- and half a step of the output's own type.
"""
import torch

STEPS = 256
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}     # half a subnormal step


def bound(mag, value, dtype):
    """Largest error of an output of ``dtype`` that rounding explains."""
    e = STEPS * 2.0 ** -24 * mag
    return e + HALF[dtype] * (value.abs() + e) + TINY[dtype]


def to_rows(t, layout):
    """[B, L, C] in float64 on the CPU."""
    t = t.detach().double().cpu()
    if layout == "nhwc":
        return t.reshape(t.shape[0], -1, t.shape[-1])
    return t.reshape(t.shape[0], t.shape[1], -1).permute(1, 2, 0)


def from_rows(t, shape, layout):
    return t.reshape(shape) if layout == "nhwc" else t.permute(2, 0, 1).reshape(shape)


def reference(x, groups, w, b, act, slope, eps, layout, gy=None, v=None, cw=None, cb=None, cs=None):
    shape = x.shape
    x = to_rows(x, layout)
    B, L, C = x.shape
    G = groups

    def par(t, none):
        t = torch.full((C,), none, dtype=torch.float64) if t is None else t.detach().double().cpu()
        return t.reshape(1, 1, G, C // G)

    def grouped(t):
        return t.reshape(B, L, G, C // G)

    def over(t):
        return t.mean((1, 3), keepdim=True)

    def chan(t):
        return t.sum((0, 1)).reshape(C)

    def data(t):
        return from_rows(t.reshape(B, L, C), shape, layout)

    w, b = par(w, 1.0), par(b, 0.0)
    x = grouped(x)
    d = x - over(x)
    r = 1 / torch.sqrt(over(d * d) + eps)
    xh = d * r
    z = xh * w + b
    mz = (xh * w).abs() + b.abs()
    a2 = torch.zeros_like(z)
    neg = z <= 0
    if act == "silu":
        s = torch.sigmoid(z)
        y, a1, a2 = z * s, s * (1 + z * (1 - s)), s * (1 - s) * (2 + z * (1 - 2 * s))
        k = torch.ones(1, dtype=torch.float64)
        ma = 1 + mz            # an error of z moves a' and a'' by less than as much
        mk = ma
    else:
        k = par(slope, 0.0) if act == "prelu" else torch.tensor(1.0 if act == "none" else float(slope),
                                                                 dtype=torch.float64)
        a1 = torch.where(neg, k.expand_as(z), torch.ones_like(z))
        y = a1 * z
        ma, mk = torch.clamp(k.abs(), min=1.0).expand_as(z), torch.zeros_like(z)
    out = {"y": (data(y), data(mz * ma))}
    if gy is None:
        return out
    gy = grouped(to_rows(gy, layout))
    g, gm = gy * a1, gy.abs() * ma
    u, um = g * w, gm * w.abs()
    mux, mmux = over(u * xh), over(um * xh.abs())
    out["gx"] = (data(r * (u - over(u) - xh * mux)), data(r * (um + over(um) + xh.abs() * mmux)))
    out["gw"] = (chan(g * xh), chan(gm * xh.abs()))
    out["gb"] = (chan(g), chan(gm))
    out["gs"] = (chan(gy * torch.where(neg, z, torch.zeros_like(z))), chan(gy.abs() * mz))
    if v is None:
        return out
    v = grouped(to_rows(v, layout))
    cs_ = par(cs, 0.0)
    cw_, cb_ = par(cw, 0.0), par(cb, 0.0)
    mvx, mmvx = over(v * xh), over((v * xh).abs())
    q, qm = r * (v - over(v) - xh * mvx), r * (v.abs() + over(v.abs()) + xh.abs() * mmvx)
    h, hm = w * q + cw_ * xh + cb_, w.abs() * qm + (cw_ * xh).abs() + cb_.abs()
    zn = torch.where(neg, z, torch.zeros_like(z))
    out["g_gy"] = (data(a1 * h + cs_ * zn), data(ma * hm + cs_.abs() * mz))
    t = gy * a2 * h + cs_ * torch.where(neg, gy, torch.zeros_like(gy))
    tm = gy.abs() * mk * hm + (cs_ * gy).abs()
    e = t * w + g * cw_ - r * (v * mux + u * mvx)
    em = tm * w.abs() + gm * cw_.abs() + r * (v.abs() * mmux + um * mmvx)
    g_x = r * (e - over(e) - xh * over(e * xh)) - r * xh * over(u * q)
    g_xm = r * (em + over(em) + xh.abs() * over(em * xh.abs())) + r * xh.abs() * over(um * qm)
    out["g_x"] = (data(g_x), data(g_xm))
    out["g_w"] = (chan(g * q + t * xh), chan(gm * qm + tm * xh.abs()))
    out["g_b"] = (chan(t), chan(tm))
    out["g_s"] = (chan(torch.where(neg, gy * h, torch.zeros_like(gy))), chan(gy.abs() * hm))
    return out


def close(got, ref, what):
    """``got`` lies within ``bound`` of the pair ``ref``."""
    value, mag = ref
    g = got.detach().double().cpu().reshape(value.shape)
    lim = bound(mag, value, got.dtype)
    err = (g - value).abs()
    bad = ~(err <= lim)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                                 f"{float((err / lim.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} bounds")
