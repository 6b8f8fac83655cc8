"""The gated feed-forward block, the norm over groups of channels and the 8-bit product, in float64 on the CPU: the definitions, and
for the rounding errors of a float32 or bfloat16 evaluation a bound of each result, carried along from the absolute values of
its terms.

Units: u = 2^-24 (half a step of float32), r = 2^-8 for bfloat16 and u for float32 (the rounding of a result). What is kept between two
products is off by r^2 = 2^-16 in bfloat16 (two parts, each rounded once) and u in float32.
A sum of n terms in float32 is off by at most (n u) times the sum of their absolute values, in any order."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
# largest |act'| and |act''|
SLOPES = {None: (1.0, 0.0), "silu": (1.1, 0.5), "gelu": (1.13, 0.8), "relu": (1.0, 0.0)}


def act(z, name):
    """The activation and its derivative."""
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    return z, torch.ones_like(z)


def rounding(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else U


def _sum(n, dtype):
    """Units of a product's sum of n terms. float32: six plane products, each term cut at 3 u of itself. bfloat16: exact terms."""
    return (6 * n + 4) * U if dtype == torch.float32 else (n + 1) * U


def gated(x, wg, wu, wd, name, gy=None):
    """[(value, bound)] of y, and for gy of the gradients of x, wg, wu, wd."""
    dtype, r = x.dtype, rounding(x.dtype)
    kept = r * r if dtype == torch.bfloat16 else r
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    first, second = SLOPES[name]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = (_sum(x.shape[1], dtype) * (x.abs() @ w.abs().T) for w in (wg, wu))
    a, d = act(g, name)
    ea = first * eg + 8 * U * (1 + g.abs())
    ed = second * eg + 16 * U * (1 + g.abs())
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + kept * h.abs()
    y = h @ wd.T
    out = [(y, eh @ wd.abs().T + _sum(h.shape[1], dtype) * (h.abs() @ wd.abs().T) + r * y.abs())]
    if gy is None:
        return out
    gy = gy.double()
    gh = gy @ wd
    egh = _sum(gy.shape[1], dtype) * (gy.abs() @ wd.abs())
    dg, du = gh * u * d, gh * a
    edg = (egh * (u * d).abs() + (gh * d).abs() * eu + (gh * u).abs() * ed) * 1.01 + kept * dg.abs()
    edu = (egh * a.abs() + gh.abs() * ea) * 1.01 + kept * du.abs()
    gx = dg @ wg + du @ wu
    terms = dg.abs() @ wg.abs() + du.abs() @ wu.abs()
    out.append((gx, edg @ wg.abs() + edu @ wu.abs() + _sum(2 * h.shape[1], dtype) * terms + r * gx.abs()))
    for left, e, right, er in ((dg, edg, x, None), (du, edu, x, None), (gy, None, h, eh)):
        v = left.T @ right
        bound = _sum(x.shape[0], dtype) * (left.abs().T @ right.abs()) + r * v.abs()
        bound = bound + (e.T @ right.abs() if er is None else left.abs().T @ er)
        out.append((v, bound))
    return out


def group_norm(x, groups, weight, bias, offsets=None, eps=1e-5, name=None, gy=None):
    """[(value, bound)] of y, and for gy of the gradients of x, weight and bias."""
    r = rounding(x.dtype)
    x = x.double()
    rows, channels = x.shape
    w = torch.ones(channels).double() if weight is None else weight.double()
    b = torch.zeros(channels).double() if bias is None else bias.double()
    first, second = SLOPES[name]
    width = channels // groups
    y, gx = torch.zeros_like(x), torch.zeros_like(x)
    ey, egx = torch.zeros_like(x), torch.zeros_like(x)
    gw, gb, egw, egb = (torch.zeros(channels).double() for _ in range(4))
    blocks = [[i, i + 1] for i in range(rows)] if offsets is None else [[int(p), int(q)] for p, q in zip(offsets[:-1], offsets[1:])]
    for p, q in blocks:
        if q <= p:
            continue
        v = x[p:q].view(q - p, groups, width)
        n = v.shape[0] * width
        k = 100 * U  # of a sum: at most 64 values in a run, then a tree, or at most 32 a lane for a row's
        mean = v.mean((0, 2), keepdim=True)
        sigma = torch.sqrt(((v - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        em = (k * v.abs().mean((0, 2), keepdim=True) + 2 * U * v.abs()) / sigma
        h = (v - mean) / sigma
        eh = em * (1 + h.abs()) + h.abs() * (k + 2 * em.mean((0, 2), keepdim=True))
        h, eh = h.reshape(-1, channels), eh.reshape(-1, channels)
        z = h * w + b
        ez = eh * w.abs() + 4 * U * ((h * w).abs() + b.abs())
        a, d = act(z, name)
        ea = first * ez + 8 * U * (1 + z.abs())
        y[p:q], ey[p:q] = a, ea + r * a.abs()
        if gy is None:
            continue
        g = gy[p:q].double()
        gz = g * d
        egz = g.abs() * (second * ez + 16 * U * (1 + z.abs()))
        runs = 64 + 2 * rows / 32 + 100
        gw, egw = gw + (gz * h).sum(0), egw + (gz.abs() * eh + egz * (h.abs() + eh) + runs * U * (gz * h).abs()).sum(0)
        gb, egb = gb + gz.sum(0), egb + (egz + runs * U * gz.abs()).sum(0)
        shape = (-1, groups, width)
        gn, egn, hh, eh3 = (gz * w).view(shape), (egz * w.abs() + U * (gz * w).abs()).view(shape), h.view(shape), eh.view(shape)
        s, t = gn.mean((0, 2), keepdim=True), (gn * hh).mean((0, 2), keepdim=True)
        es = (egn + 3 * k * gn.abs()).mean((0, 2), keepdim=True)
        et = (egn * hh.abs() + gn.abs() * eh3 + 3 * k * (gn * hh).abs()).mean((0, 2), keepdim=True) * 1.01
        total = gn.abs() + s.abs() + (hh * t).abs()
        e = (egn + es + hh.abs() * et + eh3 * t.abs() + (8 * U + k + 2 * em.mean((0, 2), keepdim=True)) * total) * 1.01
        gx[p:q] = ((gn - s - hh * t) / sigma).reshape(-1, channels)
        egx[p:q] = (e / sigma).reshape(-1, channels)
    if gy is None:
        return [(y, ey)]
    return [(y, ey), (gx, egx + r * gx.abs()), (gw, egw + r * gw.abs()), (gb, egb + r * gb.abs())]


def quantize(x):
    """(values as float64, scales float32): the definition's products and quotients are float32."""
    x = x.float()
    top = x.abs().amax(1) if x.shape[1] else x.new_zeros(x.shape[0])
    scale = top * torch.tensor(1.0 / 127.0, dtype=torch.float32)
    q = torch.round(x / torch.where(scale == 0, torch.ones_like(scale), scale)[:, None])
    return q.clamp(-127, 127).double(), scale


def linear_int8(q, scale, w, w_scale, bias, dtype):
    """(value, bound): an exact sum, its rounding, two products, the bias."""
    s = (q @ w.double().T) * scale.double()[:, None] * w_scale.double()
    y = s if bias is None else s + bias.double()
    return y, 4 * U * s.abs() + (U * y.abs() if bias is not None else 0) + rounding(dtype) * y.abs()


def near(got, want, bound, what=""):
    """Every value within its bound."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    if got.numel():
        worst = float(((got - want).abs() / (bound * 1.001 + 1e-30)).max())
        assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"
