"""Performance cases of the attention operators: what a model with attention between the atoms of a system, the
neighbours of an atom or the tokens of a sequence runs, through the framework's public entry points.

Kinds of case (``case["kind"]``):

* ``attend``  attention of the query rows of each segment over the key rows of the same segment, segments given by
              offsets: a batch of systems or sequences of different lengths (``q_rows == k_rows``), one query per
              segment over its rows (``q_rows == segments``: a readout token per system, an atom over its
              neighbours, the next token of a sequence), or other query and key counts. ``train``: with the
              gradients of queries, keys and values.
* ``norm``    the norm of queries and keys over each head with the position rotation, on the query and key columns
              of one projection. ``train``: with the gradients of both and of the two weights.

Features are standard normal (queries half as large again, for weights that are neither flat nor one-hot).
Lengths are part of the case: the same for all segments or drawn log-normally, the first two then empty and of one
row. ``exact`` is the definition in float64, segment by segment.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
BASE = 10000.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------- cases


def _attend(name, dtype, segments, q_rows, k_rows, heads, kv_heads, dim, *, ragged=False, causal=False, train=False):
    return {"name": name, "kind": "attend", "type": dtype, "segments": segments, "q_rows": q_rows, "k_rows": k_rows,
            "ragged": ragged, "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal, "train": train}


def _norm(name, dtype, rows, heads, kv_heads, dim, rot, *, interleaved=False, train=False):
    return {"name": name, "kind": "norm", "type": dtype, "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "interleaved": interleaved, "train": train}


def listed():
    return [
        # a readout token for each of eight small systems: latency of the smallest call
        _attend("readout_8x135", "f32", 8, 8, 1080, 4, 4, 32),
        # the next token of sixteen long sequences, shared key heads: one read of a long cache
        _attend("token_16x40000", "bf16", 16, 16, 640000, 16, 4, 128),
        # every atom of the headline system over its neighbours, with the gradients that the forces need
        _attend("neighbours_10000", "f32", 10000, 10000, 180096, 4, 4, 32, ragged=True, train=True),
        # all atoms of the smallest system, 128 channels: too little work to fill the card
        _attend("system_135", "f32", 1, 135, 135, 4, 4, 32),
        # a batch of systems of different sizes in one launch
        _attend("systems_16875", "f32", 16, 16875, 16875, 4, 4, 32, ragged=True),
        # the headline system's atoms, every one over all others
        _attend("system_10000", "bf16", 1, 10000, 10000, 8, 8, 64),
        # whole prompts packed one after the other, causal, shared key heads
        _attend("prompts_12000", "bf16", 5, 12000, 12000, 16, 4, 128, ragged=True, causal=True),
        # a training step's attention over a few systems in float32
        _attend("train_systems_5000", "f32", 5, 5000, 5000, 4, 4, 64, ragged=True, train=True),
        # and over packed sequences in bfloat16, causal, shared key heads
        _attend("train_packed_8192", "bf16", 4, 8192, 8192, 16, 4, 128, ragged=True, causal=True, train=True),
        # queries and keys of the smallest system: latency
        _norm("norm_135", "f32", 135, 4, 4, 32, 32),
        # queries and keys of a large batch, rotation over half of the head, neighbouring pairs
        _norm("norm_40000", "bf16", 40000, 16, 4, 128, 64, interleaved=True),
        # a training step's norm and rotation
        _norm("train_norm_16875", "f32", 16875, 8, 8, 64, 64, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = max(work(c)["flops"] for c in listed() if c["kind"] == "attend")
    while True:
        dtype = rng.choice(("f32", "bf16"))
        dim = rng.choice((16, 32, 40, 64, 96, 128))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 1, 2, 3, 4))
        train = rng.random() < 0.4
        kind = rng.choice(("norm", "self", "self", "single", "neighbours", "cross"))
        if kind == "norm":
            return _unnamed(_norm("", dtype, _log(rng, 8, 40000), heads, kv_heads, dim,
                                  2 * rng.randint(1, dim // 2), interleaved=rng.random() < 0.5, train=train))
        if kind == "single":
            segments = _log(rng, 1, 64)
            case = _attend("", dtype, segments, segments, segments * _log(rng, 16, 40000), heads, kv_heads, dim,
                           ragged=rng.random() < 0.5)
        elif kind == "neighbours":
            segments = _log(rng, 100, 10000)
            case = _attend("", dtype, segments, segments, segments * rng.randint(6, 30) + rng.randint(0, 99), heads,
                           kv_heads, dim, ragged=True, train=train)
        elif kind == "self":
            segments = _log(rng, 1, 16)
            rows = segments * _log(rng, 40, 8000) + rng.randint(0, 9)
            case = _attend("", dtype, segments, rows, rows, heads, kv_heads, dim, ragged=rng.random() < 0.7,
                           causal=rng.random() < 0.5, train=train)
        else:
            segments = _log(rng, 1, 8)
            case = _attend("", dtype, segments, segments * _log(rng, 2, 400) + 1, segments * _log(rng, 16, 8000) + 3,
                           heads, kv_heads, dim, ragged=rng.random() < 0.5, causal=rng.random() < 0.5, train=train)
        w, padded = work(case), _padded(case)
        if w["flops"] <= most and w["bytes"] <= 2 ** 30 and padded <= 2 ** 30 * (0.5 if train else 1):
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


def _case_lengths(case):
    """(query rows, key rows) of each segment."""
    lk = _lengths(case["k_rows"], case["segments"], case["ragged"])
    if case["q_rows"] == case["k_rows"]:
        return lk, lk
    return _lengths(case["q_rows"], case["segments"], case["ragged"] and case["q_rows"] != case["segments"]), lk


def _padded(case):
    """Scores of the plain form, which pads every segment to the longest."""
    lq, lk = _case_lengths(case)
    return case["segments"] * case["heads"] * max(lq) * max(lk)


def _pairs(nq, nk, causal):
    """Query-key pairs of a segment; causal: query i of nq sees the keys up to i + nk - nq."""
    if not causal:
        return nq * nk
    first = max(0, nq - nk)  # rows before it see nothing
    n = nq - first
    return n * (nk - nq + first + 1) + n * (n - 1) // 2


def work(case):
    size = 4 if case["type"] == "f32" else 2
    d, h, hk, train = case["dim"], case["heads"], case["kv_heads"], case["train"]
    if case["kind"] == "norm":
        rows = case["rows"]
        return {"bytes": rows * (h + hk) * d * size * (5 if train else 2) + rows * (case["rot"] * 4 + 4),
                "flops": rows * (h + hk) * d * (30 if train else 10)}
    lq, lk = _case_lengths(case)
    pairs = sum(_pairs(a, b, case["causal"]) for a, b in zip(lq, lk))
    q, kv = case["q_rows"] * h * d * size, case["k_rows"] * hk * d * size
    # read q, k, v (and the output's gradient), write the output (and three gradients)
    return {"bytes": 4 * q + 4 * kv if train else 2 * q + 2 * kv, "flops": pairs * h * d * (14 if train else 4)}


# ---------------------------------------------------------------------------------------- state


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)


def _offsets(lengths):
    off = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    torch.cumsum(torch.tensor(lengths, dtype=torch.int64), 0, out=off[1:])
    return off.to(DEVICE)


def _tables(positions, rot):
    """cos and sin [positions, rot / 2] of the rotation angles, formed in float64."""
    freq = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = _generator(seed)
    dtype, d, h, hk = TYPES[case["type"]], case["dim"], case["heads"], case["kv_heads"]
    s = dict(case)
    if case["kind"] == "norm":
        rows = case["rows"]
        # the projection of a block: query, key and value columns side by side
        qkv = _normal(g, rows, h + 2 * hk, d, dtype=dtype, scale=2.0)
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + hk]
        s["wq"] = (1.0 + 0.2 * torch.randn(d, generator=g, device=DEVICE)).to(dtype)
        s["wk"] = (1.0 + 0.2 * torch.randn(d, generator=g, device=DEVICE)).to(dtype)
        s["cos"], s["sin"] = _tables(max(1, rows // 2), case["rot"])
        # positions of packed sequences: each starts anew
        s["positions"] = torch.arange(rows, device=DEVICE, dtype=torch.int32) % max(1, rows // 2)
        if case["train"]:
            s["gq"], s["gk"] = _normal(g, rows, h, d, dtype=dtype), _normal(g, rows, hk, d, dtype=dtype)
        return s
    lq, lk = _case_lengths(case)
    s["max_q"], s["max_k"] = max(lq), max(lk)
    s["k_offsets"] = _offsets(lk)
    s["q_offsets"] = s["k_offsets"] if lq is lk else _offsets(lq)
    s["q"] = _normal(g, case["q_rows"], h, d, dtype=dtype, scale=1.5)
    s["k"] = _normal(g, case["k_rows"], hk, d, dtype=dtype)
    s["v"] = _normal(g, case["k_rows"], hk, d, dtype=dtype)
    if case["train"]:
        s["g"] = _normal(g, case["q_rows"], h, d, dtype=dtype)
    return s


# ---------------------------------------------------------------------------------------- passes


def run(s):
    if s["kind"] == "norm":
        return _run_norm(s) if own else _plain_norm(s)
    return _run_attend(s) if own else _plain_attend(s)


def _run_norm(s):
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, qk_norm_rotary_vjp

    args = (s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    kw = {"eps": EPS, "interleaved": s["interleaved"]}
    out = qk_norm_rotary(*args, **kw)
    if not s["train"]:
        return out
    return (*out, *qk_norm_rotary_vjp(s["gq"], s["gk"], *args, **kw))


def _run_attend(s):
    from fastmd_amd.ops.attention import segment_attention, segment_attention_forward, segment_attention_vjp

    args, offsets = (s["q"], s["k"], s["v"]), (s["q_offsets"], s["k_offsets"])
    if not s["train"]:
        return segment_attention(*args, *offsets, causal=s["causal"])
    out, lse = segment_attention_forward(*args, *offsets, causal=s["causal"])
    return (out, *segment_attention_vjp(s["g"], *args, out, lse, *offsets, causal=s["causal"]))


def _rotate(x, cos, sin, interleaved):
    """The rotation of the first columns of x [rows, heads, dim]; the transposed one for -sin."""
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    c, t = cos[:, None], sin[:, None]
    turned = torch.stack((a * c - b * t, b * c + a * t), -1)
    turned = turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def _plain_norm(s):
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    out, grads, weights = [], [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        xf, wf = x.float(), w.float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
        n = xf * r
        out.append(_rotate(n * wf, cos, sin, s["interleaved"]).to(x.dtype))
        if s["train"]:
            gy = _rotate(g.float(), cos, -sin, s["interleaved"])
            weights.append((gy * n).sum((0, 1)).to(w.dtype))
            gn = gy * wf
            grads.append((r * (gn - n * (gn * n).mean(-1, keepdim=True))).to(x.dtype))
    return (*out, *grads, *weights)


def _pad_rows(offsets, longest, rows):
    """Row of each (segment, place), clamped, and whether the place exists."""
    at = offsets[:-1, None] + torch.arange(longest, device=offsets.device)
    return at.clamp(max=rows - 1), at < offsets[1:, None]


def _unpad(x, offsets, rows, dtype):
    """[segments, kv_heads, group, places, dim] back to rows [rows, heads, dim]."""
    row = torch.arange(rows, device=offsets.device)
    seg = torch.searchsorted(offsets[1:], row, right=True)
    x = x.permute(0, 3, 1, 2, 4).flatten(2, 3)
    return x[seg, row - offsets[seg]].to(dtype)


def _plain_attend(s):
    q, k, v, qo, ko = s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"]
    (tq, h, d), (tk, hk, _) = q.shape, k.shape
    segments, group, nq, nk = s["segments"], h // hk, s["max_q"], s["max_k"]
    scale = d ** -0.5
    qi, q_is = _pad_rows(qo, nq, tq)
    ki, k_is = _pad_rows(ko, nk, tk)

    def queries(x):  # [segments * kv_heads, group * places, dim]
        x = x.float()[qi] * q_is[..., None, None]
        return x.view(segments, nq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(segments * hk, group * nq, d)

    def keys(x):  # [segments * kv_heads, places, dim]
        x = x.float()[ki] * k_is[..., None, None]
        return x.permute(0, 2, 1, 3).reshape(segments * hk, nk, d)

    qp, kp, vp = queries(q), keys(k), keys(v)
    seen = q_is[:, :, None] & k_is[:, None, :]
    if s["causal"]:
        last = torch.arange(nq, device=q.device) + ((ko[1:] - ko[:-1]) - (qo[1:] - qo[:-1]))[:, None]
        seen = seen & (torch.arange(nk, device=q.device) <= last[:, :, None])
    scores = (torch.bmm(qp, kp.transpose(1, 2)) * scale).view(segments, hk, group, nq, nk)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del scores
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, torch.ones_like(total), total)).view(segments * hk, group * nq, nk)
    op = torch.bmm(p, vp)
    shape = (segments, hk, group, nq, d)
    out = _unpad(op.view(shape), qo, tq, q.dtype)
    if not s["train"]:
        return out
    gp = queries(s["g"])
    gv = torch.bmm(p.transpose(1, 2), gp)
    gs = torch.bmm(gp, vp.transpose(1, 2))
    gs = p * (gs - (gp * op).sum(-1, keepdim=True)) * scale
    del p
    gq = torch.bmm(gs, kp)
    gk = torch.bmm(gs.transpose(1, 2), qp)
    kshape = (segments, hk, 1, nk, d)
    return (out, _unpad(gq.view(shape), qo, tq, q.dtype), _unpad(gk.view(kshape), ko, tk, q.dtype),
            _unpad(gv.view(kshape), ko, tk, q.dtype))


# ---------------------------------------------------------------------------------------- float64


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["kind"] == "norm" else _exact_attend(s)


def _exact_norm(s):
    """Complex multiplication of the weighted, normalised pairs; gradients from its adjoint."""
    pos = s["positions"].long()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    half = turn.shape[-1]
    d = s["dim"]
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + half)

    def turned(x, by):
        z = torch.complex(x.index_select(-1, first), x.index_select(-1, second)) * by
        y = x.clone()
        y.index_copy_(-1, first, z.real.contiguous())
        y.index_copy_(-1, second, z.imag.contiguous())
        return y

    out, grads, weights = [], [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        x, w = x.double(), w.double()
        rms = ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt()
        out.append(turned(x / rms * w, turn))
        if s["train"]:
            gy = turned(g.double(), turn.conj())
            weights.append((gy * x / rms).sum((0, 1)))
            gw = gy * w
            grads.append(gw / rms - x * (gw * x).sum(-1, keepdim=True) / (d * rms ** 3))
    return (*out, *grads, *weights)


def _exact_attend(s):
    """The definition for the segments of one pair of lengths together, some heads and query rows at a time."""
    lq, lk = _case_lengths(s)
    q, k, v = s["q"], s["k"], s["v"]
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    q0, k0 = s["q_offsets"].tolist(), s["k_offsets"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    gq, gk, gv = out.clone(), torch.zeros(k.shape, dtype=torch.float64, device=DEVICE), None
    gv = gk.clone()
    groups = {}
    for n, pair in enumerate(zip(lq, lk)):
        groups.setdefault(pair, []).append(n)
    for (nq, nk), members in groups.items():
        if nq == 0 or nk == 0:
            continue
        at_q = torch.tensor([q0[n] for n in members], device=DEVICE)[:, None] + torch.arange(nq, device=DEVICE)
        at_k = torch.tensor([k0[n] for n in members], device=DEVICE)[:, None] + torch.arange(nk, device=DEVICE)
        step = max(1, min(nq, 2 ** 27 // (nk * len(members))))
        for head in range(h):
            kh, vh = k[:, head // (h // hk)][at_k].double(), v[:, head // (h // hk)][at_k].double()
            sum_k, sum_v = torch.zeros_like(kh), torch.zeros_like(vh)
            for a in range(0, nq, step):
                rows = at_q[:, a:a + step]
                qh = q[:, head][rows].double()
                e = torch.matmul(qh, kh.transpose(1, 2).contiguous()) / math.sqrt(d)
                if s["causal"]:
                    i = torch.arange(a, a + rows.shape[1], device=DEVICE)[:, None] + nk - nq
                    hidden = torch.arange(nk, device=DEVICE)[None] > i
                    e.masked_fill_(hidden, -math.inf)
                p = torch.softmax(e, -1).nan_to_num_(0.0)  # a row that sees nothing gives nothing
                del e
                o = torch.matmul(p, vh)
                out[rows, head] = o
                if s["train"]:
                    gh = s["g"][:, head][rows].double()
                    sum_v += torch.matmul(p.transpose(1, 2).contiguous(), gh)
                    gp = torch.matmul(gh, vh.transpose(1, 2).contiguous())
                    gs = p * (gp - (gp * p).sum(-1, keepdim=True)) / math.sqrt(d)
                    gq[rows, head] = torch.matmul(gs, kh)
                    sum_k += torch.matmul(gs.transpose(1, 2).contiguous(), qh)
            if s["train"]:
                gk[at_k, head // (h // hk)] += sum_k
                gv[at_k, head // (h // hk)] += sum_v
    return (out, gq, gk, gv) if s["train"] else out
