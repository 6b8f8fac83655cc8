"""Performance cases of the operators between the attention layers: what a block of an attention model runs on the rows of
its atoms or tokens besides attention, through the framework's public entry points.

Kinds of case (``case["kind"]``):

* ``gated``  the gated feed-forward block ``(act(x Wg^T) * (x Wu^T)) Wd^T`` on rows [rows, width], hidden width ``hidden``.
             ``grad``: "none" (the result), "input" (with the gradient of x, as forces need), "all" (a training step).
* ``norm``   the norm over groups of channels (channels last) with its activation. ``segments`` 0: every row by itself;
             otherwise the statistics of a group are over the rows of a segment (an atom system, a map of a batch), given by
             offsets, with ``spare`` unused rows behind the last one. ``grad``: "none" or "all" (x, weight and bias).
* ``int8``   the product of rows with a weight held in 8-bit integers with a scale for each output channel; the rows are
             rounded to 8 bits on the way, with a scale for each.

Features are standard normal; in ``norm`` with a mean of their own per channel, and rows of ``int8`` differ in size as
activations do. Lengths are part of the case: the same for all segments, or drawn log-normally, the first two then empty and
of one row. ``exact`` is the definition in float64.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------- cases


def _gated(name, dtype, rows, width, hidden, *, grad="none", activation="silu", strided=False):
    return {"name": name, "kind": "gated", "type": dtype, "rows": rows, "width": width, "hidden": hidden, "grad": grad,
            "activation": activation, "strided": strided}


def _norm(name, dtype, rows, channels, groups, *, segments=0, ragged=False, spare=0, grad="none", activation="silu"):
    return {"name": name, "kind": "norm", "type": dtype, "rows": rows, "channels": channels, "groups": groups,
            "segments": segments, "ragged": ragged, "spare": spare, "grad": grad, "activation": activation}


def _int8(name, dtype, rows, width, out):
    return {"name": name, "kind": "int8", "type": dtype, "rows": rows, "width": width, "out": out}


def listed():
    return [
        # the block of the smallest system at the attention model's own widths, with what forces need: latency
        _gated("forces_135", "f32", 135, 64, 128, grad="input"),
        # the same for the headline system
        _gated("forces_10000", "f32", 10000, 64, 128, grad="input"),
        # a training step of a wider model over a union of systems, float32, a hidden width of 8/3
        _gated("train_16875", "f32", 16875, 256, 680, grad="all"),
        # the next token of sixteen sequences: one read of the weights
        _gated("token_16", "bf16", 16, 2048, 5504),
        # whole prompts, packed
        _gated("prompts_12000", "bf16", 12000, 1024, 2736),
        # a training step over packed sequences
        _gated("train_8192", "bf16", 8192, 2048, 5504, grad="all"),
        # every atom of the smallest system by itself: latency
        _norm("norm_135", "f32", 135, 64, 4),
        # a training step's norm over systems of different sizes in one buffer with unused rows behind them
        _norm("train_systems_16875", "f32", 16875, 128, 8, segments=16, ragged=True, spare=509, grad="all"),
        # maps of a batch, channels last: 64 x 64 places of 320 channels
        _norm("maps_16x4096", "bf16", 65536, 320, 32, segments=16),
        # a training step over larger maps of fewer channels
        _norm("train_maps_16x16384", "bf16", 262144, 128, 32, segments=16, grad="all"),
        # the next token of sixteen sequences through 8-bit weights
        _int8("int8_token_16", "bf16", 16, 4096, 4096),
        # a long packed batch through them
        _int8("int8_8192", "bf16", 8192, 4096, 4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most_flops = max(work(c)["flops"] for c in listed())
    most_bytes = max(work(c)["bytes"] for c in listed() if c["kind"] == "norm")
    while True:
        dtype = rng.choice(("f32", "bf16"))
        # without "relu" where there are gradients: which side of its step a value near 0 is on is a matter of its last bit
        smooth = rng.choice(("silu", "silu", "gelu"))
        sharp = rng.choice((smooth, smooth, "relu"))
        kind = rng.choice(("gated", "gated", "gated", "norm", "norm", "int8"))
        if kind == "gated":
            width = _log(rng, 16, 2048)
            hidden = int(width * rng.uniform(1.3, 4.0))
            if rng.random() < 0.7:  # most widths are whole vectors
                width, hidden = -(-width // 8) * 8, -(-hidden // 8) * 8
            grad = rng.choice(("none", "input", "all"))
            case = _gated("", dtype, _log(rng, 1, 12000), width, hidden, grad=grad,
                          activation=sharp if grad == "none" else smooth, strided=rng.random() < 0.3)
            if work(case)["flops"] <= most_flops * (1.0 if dtype == "bf16" else 0.25):
                return _unnamed(case)
        elif kind == "norm":
            groups = rng.choice((1, 2, 4, 8, 16, 32))
            segments = 0 if rng.random() < 0.35 else _log(rng, 1, 300)
            # a mean of a few values takes most of them away, and their gradients with it: 8 in a row, 16 in a segment
            width = _log(rng, 1 if segments else 8, max(8, 640 // groups))
            channels, rows = groups * width, max(1, segments) * _log(rng, 16 // min(width, 16), 16384) + rng.randint(0, 9)
            grad = rng.choice(("none", "all"))
            case = _norm("", dtype, rows, channels, groups, segments=segments, ragged=rng.random() < 0.6,
                         spare=rng.choice((0, 0, 1, 37)) if segments else 0, grad=grad,
                         activation=rng.choice((sharp if grad == "none" else smooth, "none")))
            if work(case)["bytes"] <= most_bytes:
                return _unnamed(case)
        else:
            case = _int8("", dtype, _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 16, 8192))
            if work(case)["flops"] <= most_flops * 0.25:
                return _unnamed(case)


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(rows, segments, ragged):
    """The rows of each segment: equal to within one, or log-normal with an empty and a one-row segment in front."""
    if not ragged or segments == 1:
        return [rows // segments + (s < rows % segments) for s in range(segments)]
    rng = random.Random(rows * 1009 + segments)
    front = [0, 1] if segments > 4 else []
    weights = [math.exp(0.5 * rng.gauss(0.0, 1.0)) for _ in range(segments - len(front))]
    left, total = rows - sum(front), sum(weights)
    lengths = [int(left * w / total) for w in weights]
    for s in range(left - sum(lengths)):
        lengths[s % len(lengths)] += 1
    return front + lengths


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "norm":
        values = (case["rows"] + case["spare"]) * case["channels"]
        # read x (and the output's gradient), write the output (and the gradient)
        return {"bytes": values * size * (4 if case["grad"] == "all" else 2), "flops": values * (40 if case["grad"] == "all" else 15)}
    rows, width = case["rows"], case["width"]
    if case["kind"] == "int8":
        return {"bytes": rows * (width + case["out"]) * size + width * case["out"], "flops": 2 * rows * width * case["out"]}
    hidden, grad = case["hidden"], case["grad"]
    passes = {"none": 1, "input": 2, "all": 2}[grad]
    return {"bytes": (2 * passes * rows * width + 3 * width * hidden * (2 if grad == "all" else 1)) * size,
            "flops": rows * width * hidden * {"none": 6, "input": 12, "all": 18}[grad]}


# ---------------------------------------------------------------------------------------- state


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    dtype = TYPES[case["type"]]
    s = dict(case)
    if case["kind"] == "gated":
        rows, width, hidden = case["rows"], case["width"], case["hidden"]
        # rows of their own, or columns of a wider buffer
        s["x"] = _normal(g, rows, width + (16 if case["strided"] else 0), dtype=dtype)[:, :width]
        packed = _normal(g, 2 * hidden, width, dtype=dtype, scale=width ** -0.5)  # both projections in one matrix
        s["w_gate"], s["w_up"] = packed[:hidden], packed[hidden:]
        s["w_down"] = _normal(g, width, hidden, dtype=dtype, scale=hidden ** -0.5)
        if case["grad"] != "none":
            s["g"] = _normal(g, rows, width, dtype=dtype)
        return s
    if case["kind"] == "int8":
        rows, width, out = case["rows"], case["width"], case["out"]
        size = torch.exp(torch.randn(rows, 1, generator=g, device=DEVICE))
        s["x"] = (torch.randn(rows, width, generator=g, device=DEVICE) * size).to(dtype)
        w = torch.randn(out, width, generator=g, device=DEVICE) * width ** -0.5
        s["w_scale"] = w.abs().amax(1) / 127.0  # rounded once, when the model was loaded
        s["w"] = torch.round(w / s["w_scale"][:, None]).to(torch.int8)
        return s
    rows, channels = case["rows"], case["channels"]
    mean = torch.randn(channels, generator=g, device=DEVICE)
    s["x"] = (torch.randn(rows + case["spare"], channels, generator=g, device=DEVICE) + mean).to(dtype)
    s["weight"] = (1.0 + 0.2 * torch.randn(channels, generator=g, device=DEVICE)).to(dtype)
    s["bias"] = (0.2 * torch.randn(channels, generator=g, device=DEVICE)).to(dtype)
    s["offsets"] = None
    if case["segments"]:
        lengths = _lengths(rows, case["segments"], case["ragged"])
        offsets = torch.zeros(len(lengths) + 1, dtype=torch.int64)
        torch.cumsum(torch.tensor(lengths, dtype=torch.int64), 0, out=offsets[1:])
        s["offsets"] = offsets.to(DEVICE)
    if case["grad"] == "all":
        s["g"] = _normal(g, rows + case["spare"], channels, dtype=dtype)
    return s


# ---------------------------------------------------------------------------------------- passes


def run(s):
    kind = s["kind"]
    if own:
        return _own_gated(s) if kind == "gated" else _own_norm(s) if kind == "norm" else _own_int8(s)
    return _plain_gated(s) if kind == "gated" else _plain_norm(s) if kind == "norm" else _plain_int8(s)


def _own_gated(s):
    from fastmd_amd.ops.feed_forward import (gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp)

    args, act = (s["x"], s["w_gate"], s["w_up"], s["w_down"]), s["activation"]
    if s["grad"] == "none":
        return gated_feed_forward(*args, activation=act)
    y, saved = gated_feed_forward_forward(*args, activation=act)
    grads = gated_feed_forward_vjp(s["g"], *args, saved, activation=act, need_weights=s["grad"] == "all")
    return (y, *(x for x in grads if x is not None))


def _own_norm(s):
    from fastmd_amd.ops.group_norm import group_norm, group_norm_forward, group_norm_vjp

    act = None if s["activation"] == "none" else s["activation"]
    args, kw = (s["x"], s["groups"], s["weight"], s["bias"]), {"offsets": s["offsets"], "activation": act}
    if s["grad"] == "none":
        return group_norm(*args, eps=EPS, **kw)
    y, saved = group_norm_forward(*args, eps=EPS, **kw)
    return (y, *group_norm_vjp(s["g"], *args, saved, **kw))


def _own_int8(s):
    from fastmd_amd.ops.int8 import Int8Rows, linear_int8

    return linear_int8(s["x"], Int8Rows(s["w"], s["w_scale"]))


def _activate(z, name):
    """The activation and its derivative."""
    if name == "silu":
        t = 1.0 / (1.0 + torch.exp(-z))
        return z * t, t * (1.0 + z * (1.0 - t))
    if name == "gelu":
        t = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * t, t + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    return z, torch.ones_like(z)


def _plain_gated(s):
    dtype = s["x"].dtype
    x, wg, wu, wd = s["x"].float(), s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
    gate, up = x @ wg.T, x @ wu.T
    a, d = _activate(gate, s["activation"])
    h = a * up
    y = (h @ wd.T).to(dtype)
    if s["grad"] == "none":
        return y
    g = s["g"].float()
    gh = g @ wd
    ggate, gup = gh * up * d, gh * a
    gx = (ggate @ wg + gup @ wu).to(dtype)
    if s["grad"] == "input":
        return y, gx
    return y, gx, (ggate.T @ x).to(dtype), (gup.T @ x).to(dtype), (g.T @ h).to(dtype)


def _row_segments(offsets, rows):
    """The segment of each row, and whether it is in one."""
    row = torch.arange(rows, device=offsets.device)
    seg = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    return seg.clamp(max=offsets.shape[0] - 2), row < offsets[-1]


def _segment_sums(x, offsets):
    """Sums of x [rows, groups] over the rows of each segment: differences of running sums in 64 bits."""
    total = torch.cumsum(x.T.double().contiguous(), 1)
    total = torch.cat((torch.zeros_like(total[:, :1]), total), 1)
    return (total[:, offsets[1:]] - total[:, offsets[:-1]]).T


def _plain_norm(s):
    x, groups = s["x"], s["groups"]
    rows, channels = x.shape
    width = channels // groups
    xf = x.float().view(rows, groups, width)
    if s["offsets"] is None:
        live = None

        def mean_of(v):
            return v.mean(-1)
    else:
        seg, live = _row_segments(s["offsets"], rows)
        count = ((s["offsets"][1:] - s["offsets"][:-1]).clamp(min=1) * width)[:, None]

        def mean_of(v):
            return (_segment_sums(v.sum(-1), s["offsets"]) / count).float()[seg]

    centred = xf - mean_of(xf)[..., None]
    rstd = torch.rsqrt(mean_of(centred * centred) + EPS)[..., None]
    n = centred * rstd
    w, b = s["weight"].float().view(groups, width), s["bias"].float().view(groups, width)
    a, d = _activate(n * w + b, s["activation"])
    if live is not None:
        a = a * live[:, None, None]
    y = a.reshape(rows, channels).to(x.dtype)
    if s["grad"] == "none":
        return y
    gz = s["g"].float().view(rows, groups, width) * d
    if live is not None:
        gz = gz * live[:, None, None]
    gn = gz * w
    gx = rstd * (gn - mean_of(gn)[..., None] - n * mean_of(gn * n)[..., None])
    if live is not None:
        gx = gx * live[:, None, None]
    return (y, gx.reshape(rows, channels).to(x.dtype), (gz * n).sum(0).view(channels).to(x.dtype),
            gz.sum(0).view(channels).to(x.dtype))


def _plain_int8(s):
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127.0
    q = torch.round(x / torch.where(scale == 0, torch.ones_like(scale), scale))
    return ((q @ s["w"].float().T) * scale * s["w_scale"]).to(s["x"].dtype)


# ---------------------------------------------------------------------------------------- float64


def exact(case, seed):
    s = prepare(case, seed)
    return {"gated": _exact_gated, "norm": _exact_norm, "int8": _exact_int8}[case["kind"]](s)


def _exact_activation(z, name):
    """The activation and its derivative, the derivative by differentiation."""
    with torch.enable_grad():
        z = z.detach().requires_grad_()
        if name == "silu":
            a = z * torch.sigmoid(z)
        elif name == "gelu":
            a = z * torch.special.ndtr(z)
        elif name == "relu":
            a = torch.relu(z)
        else:
            a = z * 1.0
        (d,) = torch.autograd.grad(a.sum(), z)
    return a.detach(), d


def _exact_gated(s):
    x, wg, wu, wd = (s[k].double() for k in ("x", "w_gate", "w_up", "w_down"))
    rows = x.shape[0]
    step = max(1, 2 ** 25 // wg.shape[0])
    y = torch.empty_like(x)
    gx = torch.empty_like(x)
    sums = [torch.zeros_like(wg), torch.zeros_like(wu), torch.zeros_like(wd)]
    for a in range(0, rows, step):
        part = x[a:a + step]
        up = torch.mm(part, wu.t())
        value, slope = _exact_activation(torch.mm(part, wg.t()), s["activation"])
        y[a:a + step] = torch.mm(value * up, wd.t())
        if s["grad"] == "none":
            continue
        g = s["g"][a:a + step].double()
        gh = torch.mm(g, wd)
        down = (gh * up * slope, gh * value)
        gx[a:a + step] = torch.mm(down[0], wg) + torch.mm(down[1], wu)
        if s["grad"] == "all":
            sums[0] += torch.mm(down[0].t(), part)
            sums[1] += torch.mm(down[1].t(), part)
            sums[2] += torch.mm(g.t(), value * up)
    return y if s["grad"] == "none" else (y, gx) if s["grad"] == "input" else (y, gx, *sums)


def _exact_norm(s):
    """Segment by segment (or all rows at once, each by itself), in blocks of [segments, rows, groups, width]."""
    x, groups = s["x"].double(), s["groups"]
    rows, channels = x.shape
    w, b = s["weight"].double(), s["bias"].double()
    out, gx = torch.zeros_like(x), torch.zeros_like(x)
    gw, gb = torch.zeros_like(w), torch.zeros_like(b)
    if s["offsets"] is None:
        blocks = [(slice(a, min(rows, a + 32768)), True) for a in range(0, rows, 32768)]
    else:
        ends = s["offsets"].tolist()
        blocks = [(slice(a, z), False) for a, z in zip(ends[:-1], ends[1:]) if z > a]
    for block, alone in blocks:
        v = x[block]
        v = v.view(v.shape[0] if alone else 1, -1, groups, channels // groups)
        var, mean = torch.var_mean(v, dim=(1, 3), correction=0, keepdim=True)
        n = (v - mean) / torch.sqrt(var + EPS)
        value, slope = _exact_activation((n.reshape(-1, channels) * w + b), s["activation"])
        out[block] = value
        if s["grad"] == "all":
            gz = s["g"][block].double() * slope
            gw += (gz * n.reshape(-1, channels)).sum(0)
            gb += gz.sum(0)
            gn = (gz * w).view(v.shape)
            gn = gn - gn.mean((1, 3), keepdim=True) - n * (gn * n).mean((1, 3), keepdim=True)
            gx[block] = (gn / torch.sqrt(var + EPS)).reshape(-1, channels)
    return out if s["grad"] == "none" else (out, gx, gw, gb)


def _exact_int8(s):
    """The rounding to 8 bits is defined in float32 (a quotient, to the nearest integer); the rest in float64."""
    top = torch.linalg.vector_norm(s["x"].float(), math.inf, dim=1)
    scale = top.div(127.0)
    q = s["x"].float().div(scale.clamp(min=1e-45)[:, None]).round().double()
    return torch.mm(q, s["w"].double().t()) * scale.double()[:, None] * s["w_scale"].double()[None]
