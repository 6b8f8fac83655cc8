"""Attention within segments and the norm and rotation of its queries and keys, in float64 on the CPU: the definitions,
one segment and one head at a time, and the magnitudes that bound their rounding errors."""
from __future__ import annotations

import math

import torch


def visible(nq: int, nk: int, causal: bool) -> torch.Tensor:
    """[nq, nk]: the last query sees every key, each one before it one key less."""
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None]
    return (j <= i + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool)


def segment_attention(q, k, v, q_off, k_off, *, causal=False, scale=None, gout=None):
    """dict with out and lse (and gq, gk, gv for gout), and for each output `x` a magnitude `abs_x`: the sum of the
    absolute values of the terms that its definition adds. Keys that a query does not see are not touched for it."""
    q, k, v = q.double(), k.double(), v.double()
    (tq, h, d), (tk, hk, _) = q.shape, k.shape
    scale = d ** -0.5 if scale is None else scale
    r = {n: torch.zeros(tq, h, d, dtype=torch.float64) for n in ("out", "abs_out", "gq", "abs_gq")}
    r |= {n: torch.zeros(tk, hk, d, dtype=torch.float64) for n in ("gk", "gv", "abs_gk", "abs_gv")}
    r["lse"] = torch.full((h, tq), -math.inf, dtype=torch.float64)
    r["scores"] = 0.0  # largest sum of absolute products in a score
    g = None if gout is None else gout.double()
    q_off, k_off = [int(x) for x in q_off], [int(x) for x in k_off]
    for s in range(len(q_off) - 1):
        rows, keys = slice(q_off[s], q_off[s + 1]), slice(k_off[s], k_off[s + 1])
        nq, nk = rows.stop - rows.start, keys.stop - keys.start
        if nq <= 0 or nk <= 0:
            continue
        sees = visible(nq, nk, causal)
        live = sees.any(0)  # keys that anybody sees
        rows_live = sees.any(1)
        for a in range(h):
            b = a // (h // hk)
            kk, vv = k[keys, b].clone(), v[keys, b].clone()
            kk[~live] = 0.0
            vv[~live] = 0.0
            qq = q[rows, a]
            s_ij = (qq @ kk.T * scale).masked_fill(~sees, -math.inf)
            r["scores"] = max(r["scores"], float((qq.abs() @ kk.abs().T * scale).masked_fill(~sees, 0.0).max()))
            top = s_ij.amax(1, keepdim=True)
            e = torch.exp(s_ij - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = e.sum(1, keepdim=True)
            p = torch.where(total > 0, e / total, torch.zeros_like(e))
            o, ao = p @ vv, p @ vv.abs()
            r["out"][rows, a], r["abs_out"][rows, a] = o, ao
            r["lse"][a, rows] = torch.where(rows_live, (top + torch.log(total))[:, 0], r["lse"][a, rows])
            if g is None:
                continue
            gg = g[rows, a]
            dp, adp = gg @ vv.T, gg.abs() @ vv.abs().T
            delta, adelta = (gg * o).sum(1, keepdim=True), (gg.abs() * ao).sum(1, keepdim=True)
            ds, ads = p * (dp - delta) * scale, p * (adp + adelta) * scale
            r["gq"][rows, a], r["abs_gq"][rows, a] = ds @ kk, ads @ kk.abs()
            r["gk"][keys, b] += ds.T @ qq
            r["abs_gk"][keys, b] += ads.T @ qq.abs()
            r["gv"][keys, b] += p.T @ gg
            r["abs_gv"][keys, b] += p.T @ gg.abs()
    return r


def norm_rotary(x, weight, cos, sin, positions=None, *, eps=1e-6, interleaved=False, norm=True, g=None):
    """(y, None, None), or (y, gradient of x, of weight) for the gradient `g` of y. x [tokens, heads, dim]."""
    x = x.double().clone().requires_grad_(g is not None)
    d, half = x.shape[-1], cos.shape[1]
    w = torch.ones(d, dtype=torch.float64) if weight is None else weight.double().clone()
    w.requires_grad_(g is not None)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w if norm else x * 1.0
    rows = torch.arange(x.shape[0]) if positions is None else positions.long()
    c, s = cos.double()[rows][:, None], sin.double()[rows][:, None]
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = y[..., first], y[..., second]
    out = y.clone()
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    if g is None:
        return out, None, None
    gx, gw = torch.autograd.grad(out, (x, w), g.double(), allow_unused=True)
    return out.detach(), gx, gw
