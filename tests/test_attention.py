"""(g) Attention within segments: the HIP kernels against the definition in float64.

Error bounds (before any run). u = 2^-8 for a rounding to bf16's 8 bits, 2^-24 for float32. `abs_x` sums the absolute values of the
terms of x. Scores: a product of three-plane operands drops terms below 3 * 2^-24 of it and is added in fp32, over at most
128 columns; the score's error is below 16 * 2^-24 of its absolute sum (rounding errors of a sum of n terms grow like
sqrt(n), 11 for 128), times log2(e) and back in the exponent; an exponential's relative error is the score's error, the
instruction's 2^-22 and the same of the row sum. Together 2 * (16 * 2^-24 * S + 2^-20) for the largest absolute sum S.
bf16: scores as above (products of bf16 are exact in fp32), and
* out: p rounded (u abs_out), out rounded (u |out|);
* gv: p rounded, gv rounded;
* gq, gk: dS rounded (u), delta from the rounded output (whose own error is u abs_out + u |out| <= 2 u abs_out): 3 u in all
  of abs_gq, abs_gk; the result rounded (u).
"""
import math

import pytest
import torch

from oracle import attention as oracle

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]


def bounds(r, dtype):
    fp32 = 2.0 * (16.0 * 2.0 ** -24 * r["scores"] + 2.0 ** -20)
    u = U[dtype]
    extra = {"out": u, "gv": u, "gq": 3 * u, "gk": 3 * u} if dtype == torch.bfloat16 else dict.fromkeys(
        ("out", "gv", "gq", "gk"), 0.0)
    return {n: r["abs_" + n] * 1.01 * (fp32 + e) + 1.01 * u * r[n].abs() + 1e-30 for n, e in extra.items()}


def offsets(lengths, before=0):
    off = [before]
    for n in lengths:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int64)


def make(lq, lk, heads, kv_heads, dim, dtype, *, before=0, after=0, seed=0, scale_q=1.5):
    g = torch.Generator().manual_seed(seed)
    q_off, k_off = offsets(lq, before), offsets(lk, before)
    tq, tk = int(q_off[-1]) + after, int(k_off[-1]) + after
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    q = (torch.randn(tq, heads, dim, generator=g) * scale_q).to(dtype)
    return q, rand(tk, kv_heads, dim), rand(tk, kv_heads, dim), rand(tq, heads, dim), q_off, k_off


def compare(got, want, bound, name):
    got = got.double().cpu()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()), f"{name} is not finite"
    worst = float(((got - want).abs() / bound).max()) if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} of the bound"


def check(q, k, v, g, q_off, k_off, *, causal, scale=None, device="cuda"):
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    r = oracle.segment_attention(q, k, v, q_off, k_off, causal=causal, scale=scale, gout=g)
    b = bounds(r, q.dtype)
    d = [x.to(device) for x in (q, k, v, g, q_off, k_off)]
    out, saved = segment_attention_forward(*d[:3], *d[4:], causal=causal, scale=scale)
    lse = saved.lse
    compare(out, r["out"], b["out"], "out")
    seen = torch.isfinite(r["lse"])
    assert torch.equal(lse.cpu()[~seen], torch.full_like(lse.cpu()[~seen], -math.inf))
    if seen.any():
        # log of the sum: the scores' error, and the rounding of a result of its size
        far = (lse.cpu().double() - r["lse"])[seen].abs()
        tol = 2.0 * (16.0 * 2.0 ** -24 * r["scores"] + 2.0 ** -20) + 2.0 ** -22 * r["lse"][seen].abs()
        assert bool((far <= tol).all())
    grads = segment_attention_vjp(d[3], *d[:3], out, saved, *d[4:], causal=causal, scale=scale)
    for name, x in zip(("gq", "gk", "gv"), grads):
        compare(x, r[name], b[name], name)
    return out, lse, grads


SHAPES = [  # query lengths, key lengths (None: the same), heads, kv_heads
    ([1], None, 1, 1),
    ([135], None, 4, 4),
    ([0, 1, 31, 32, 33, 0], None, 2, 1),
    ([63, 64, 65], None, 6, 2),
    ([127, 128, 129, 2], None, 3, 3),
    ([1, 1, 1, 1], [70, 0, 1, 300], 8, 2),
    ([5, 0, 40, 7], [3, 9, 0, 100], 4, 1),
    ([300, 17], [40, 500], 2, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_lengths_and_heads(shape, dtype, causal):
    lq, lk, heads, kv_heads = SHAPES[shape]
    q, k, v, g, q_off, k_off = make(lq, lq if lk is None else lk, heads, kv_heads, 32, dtype, seed=shape)
    check(q, k, v, g, q_off, k_off, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 96, 104, 128])
def test_head_widths(dim, dtype):
    q, k, v, g, q_off, k_off = make([70, 3, 129], [70, 3, 129], 4, 2, dim, dtype, seed=dim)
    check(q, k, v, g, q_off, k_off, causal=True)
    check(q, k, v, g, q_off, k_off, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_wide_tiles(dim, dtype, causal):
    """Enough rows for the tiles of 128, with ragged ends."""
    lengths = [1100, 0, 1, 700, 2300]
    q, k, v, g, q_off, k_off = make(lengths, lengths, 8, 8, dim, dtype, seed=dim)
    check(q, k, v, g, q_off, k_off, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [16, 24, 64, 72, 128])
def test_middle_sizes_in_float32(dim, causal):
    """Enough rows for staged planes, too few for four waves of rows per tile."""
    q, k, v, g, q_off, k_off = make([900, 1, 0, 801, 700], [900, 33, 5, 801, 650], 4, 4, dim, torch.float32, seed=dim)
    check(q, k, v, g, q_off, k_off, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [16, 32])
def test_middle_sizes_of_narrow_heads_in_float32(dim, causal):
    q, k, v, g, q_off, k_off = make([1300, 1, 0, 1201, 900], [1300, 33, 5, 1201, 950], 4, 4, dim, torch.float32, seed=dim)
    check(q, k, v, g, q_off, k_off, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_many_segments_of_a_few_hundred_rows(dtype):
    """Single queries, enough segments for a wave each over longer keys."""
    g = torch.Generator().manual_seed(8)
    lk = torch.randint(100, 260, (1030,), generator=g).tolist()
    lk[3], lk[4], lk[1029] = 0, 900, 1
    q, k, v, go, q_off, k_off = make([1] * 1030, lk, 2, 1, 24, dtype, seed=9)
    check(q, k, v, go, q_off, k_off, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 128])
def test_wide_tiles_with_shared_heads_and_other_key_counts(dim, dtype):
    q, k, v, g, q_off, k_off = make([900, 1500, 33], [2000, 1300, 65], 12, 4, dim, dtype, seed=dim)
    check(q, k, v, g, q_off, k_off, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 128), (4, 4, 32), (3, 1, 96), (40, 1, 64)])
def test_single_queries_over_long_keys(heads, kv_heads, dim, dtype):
    """The key axis split over workgroups, segments of very different lengths among the splits."""
    from fastmd_amd import _abi

    lk = [6000, 1, 0, 513, 2049]
    q, k, v, g, q_off, k_off = make([1] * 5, lk, heads, kv_heads, dim, dtype, seed=dim)
    assert _abi.load().fmd_segment_attention_splits(int(dtype == torch.bfloat16), 5, sum(lk), 5, heads, kv_heads, dim) > 1
    check(q, k, v, g, q_off, k_off, causal=False)
    check(q, k, v, g, q_off, k_off, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2)])
def test_neighbour_rows(heads, kv_heads, dtype):
    """One query per segment over a few rows each: an atom over its neighbours."""
    g = torch.Generator().manual_seed(3)
    lk = torch.randint(0, 40, (700,), generator=g).tolist()
    lk[0], lk[1], lk[-1] = 0, 150, 0
    q, k, v, go, q_off, k_off = make([1] * 700, lk, heads, kv_heads, 32, dtype, before=3, after=5)
    check(q, k, v, go, q_off, k_off, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (8, 2, 16), (3, 1, 40), (10, 5, 128), (4, 2, 96), (9, 9, 64)])
def test_few_rows_of_any_group_and_width(heads, kv_heads, dim, dtype, causal):
    """Mostly single queries, some segments with none and some with several."""
    g = torch.Generator().manual_seed(dim)
    lk = torch.randint(0, 30, (300,), generator=g).tolist()
    lq = [1] * 300
    lq[5], lq[6], lq[7], lq[200], lq[201], lq[299] = 0, 4, 0, 3, 0, 0
    q, k, v, go, q_off, k_off = make(lq, lk, heads, kv_heads, dim, dtype, seed=dim)
    check(q, k, v, go, q_off, k_off, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,lk", [([60, 90], [60, 90]), ([1, 1], [200, 30]), ([1100, 1500], [1100, 1500])])
def test_rows_outside_the_segments(lq, lk, dtype):
    """Rows before the first and after the last offset: zero output and gradient, and their NaN reaches nobody."""
    q, k, v, g, q_off, k_off = make(lq, lk, 8, 8, 64, dtype, before=7, after=70)
    for x, off in ((q, q_off), (k, k_off), (v, k_off), (g, q_off)):
        x[:int(off[0])] = float("nan")
        x[int(off[-1]):] = float("nan")
    r = oracle.segment_attention(q, k, v, q_off, k_off, gout=g)
    out, lse, grads = check(q, k, v, g, q_off, k_off, causal=False)
    for x, off in zip((out, *grads), (q_off, q_off, k_off, k_off)):
        assert not x[:int(off[0])].any() and not x[int(off[-1]):].any()
    assert torch.isinf(lse[:, :7]).all()
    assert not r["out"][:7].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_values_of_other_segments_do_not_matter(dtype):
    """A segment of NaN and infinities beside finite ones (tiles run past the ends of segments)."""
    lengths = [50, 45, 61]
    q, k, v, g, q_off, k_off = make(lengths, lengths, 4, 2, 32, dtype)
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    def run(q, k, v, g):
        a = [x.cuda() for x in (q, k, v)]
        off = q_off.cuda()
        out, saved = segment_attention_forward(*a, off)
        return (out, *segment_attention_vjp(g.cuda(), *a, out, saved, off))

    want = run(q, k, v, g)
    for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (g, float("-inf"))):
        x[50:95] = bad
    got = run(q, k, v, g)
    for a, b in zip(got, want):
        assert torch.equal(a[:50], b[:50]) and torch.equal(a[95:], b[95:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([80], 2, 1, 32), ([150, 61], 4, 4, 64), ([70], 6, 2, 96), ([200], 1, 1, 128),
                                                        ([1500, 900], 16, 4, 64), ([1300, 1500], 16, 16, 32),
                                                        ([900, 1000], 4, 4, 64), ([1300, 900], 16, 4, 128),
                                                        ([1] * 300, 2, 2, 32)])
def test_rows_that_are_not_seen_yet_do_not_matter(lengths, heads, kv_heads, dim, dtype):
    """Causal, with infinities and NaN from the middle of each segment on: the rows before are as without them; and so are
    the gradients of the keys after a query's gradient that is not finite."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    q, k, v, g, off, _ = make(lengths, lengths, heads, kv_heads, dim, dtype, seed=dim)
    start = off.tolist()
    cut = [a + (b - a) // 2 + 3 for a, b in zip(start, start[1:])]
    before = torch.cat([torch.arange(a, min(c, b)) for a, c, b in zip(start, cut, start[1:])])
    after = torch.cat([torch.arange(min(c, b), b) for c, b in zip(cut, start[1:])])

    def run(q, k, v, g):
        x = [t.cuda() for t in (q, k, v, g)]
        o = off.cuda()
        out, saved = segment_attention_forward(*x[:3], o, causal=True)
        return [t.cpu() for t in (out, *segment_attention_vjp(x[3], *x[:3], out, saved, o, causal=True))]

    want = run(q, k, v, g)
    k2, v2 = k.clone(), v.clone()
    k2[after], v2[after] = float("nan"), float("inf")
    v2[after[::3]] = float("nan")
    got = run(q, k2, v2, g)
    assert torch.isfinite(got[0][before]).all() and torch.isfinite(got[1][before]).all()
    r = oracle.segment_attention(q, k, v, off, off, causal=True, gout=g)
    b = bounds(r, dtype)
    for n, name in ((0, "out"), (1, "gq")):
        compare(got[n][before], r[name][before], b[name][before], name)
    # a gradient that is not finite in the first half: the keys after it are not seen by those queries
    q2, g2 = q.clone(), g.clone()
    g2[before], q2[before[::2]] = float("nan"), float("inf")
    got = run(q2, k, v, g2)
    for n, name in ((2, "gk"), (3, "gv")):
        compare(got[n][after], r[name][after], b[name][after], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(dtype):
    """Columns of a packed projection, a head-major layout, a strided gradient, unaligned and broadcast inputs."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    lengths = [90, 40]
    q, k, v, g, off, _ = make(lengths, lengths, 4, 2, 32, dtype)
    off = off.cuda()
    q, k, v, g = (x.cuda() for x in (q, k, v, g))

    def run(q, k, v, g):
        out, saved = segment_attention_forward(q, k, v, off, causal=True)
        return (out, saved.lse, *segment_attention_vjp(g, q, k, v, out, saved, off, causal=True))

    want = run(q, k, v, g)
    packed = torch.cat((q, k, v), 1)
    head_major = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    spread = torch.empty(*q.shape, 2, dtype=dtype, device="cuda")[..., 0].copy_(q)
    for case in ((packed[:, :4], packed[:, 4:6], packed[:, 6:], g), (head_major(q), head_major(k), head_major(v),
                                                                    head_major(g)), (odd, k, v, g), (spread, k, v, g)):
        for a, b in zip(run(*case), want):
            assert torch.equal(a, b)
    one = k[:1].expand(130, 2, 32)  # a broadcast row
    for a, b in zip(run(q, one, v, g), run(q, one.contiguous(), v, g)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,lk,heads", [([135, 60], [135, 60], 4), ([1, 1], [5000, 60], 4), ([1500, 2000], [1500, 2000], 8)])
def test_runs_are_bitwise_repeatable(lq, lk, heads, dtype):
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    q, k, v, g, q_off, k_off = (x.cuda() for x in make(lq, lk, heads, heads, 32, dtype))

    def run():
        out, saved = segment_attention_forward(q, k, v, q_off, k_off)
        return (out, saved.lse, *segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off))

    for a, b in zip(run(), run()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_autograd_against_differences(causal):
    """Directional derivatives of a scalar of the float32 output by central differences in float64 of the oracle."""
    from fastmd_amd.ops.attention import segment_attention

    q, k, v, g, q_off, k_off = make([20, 33], [28, 30], 4, 2, 16, torch.float32, seed=5)
    a = [x.cuda().requires_grad_() for x in (q, k, v)]
    out = segment_attention(*a, q_off.cuda(), k_off.cuda(), causal=causal)
    (out * g.cuda()).sum().backward()
    gen = torch.Generator().manual_seed(9)
    for n in range(3):
        way = torch.randn(a[n].shape, generator=gen).double()
        value = []
        for step in (1e-4, -1e-4):
            x = [t.double() for t in (q, k, v)]
            x[n] = x[n] + step * way
            value.append(float((oracle.segment_attention(*x, q_off, k_off, causal=causal)["out"] * g.double()).sum()))
        want = (value[0] - value[1]) / 2e-4
        got = float((a[n].grad.double().cpu() * way).sum())
        # truncation of the differences: step^2 times third derivatives of order one per term
        assert abs(got - want) <= 1e-5 * float((a[n].grad.double().cpu() * way).abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """Scores of several hundred: the running maximum keeps every exponential finite."""
    q, k, v, g, q_off, k_off = make([70, 200], [70, 200], 2, 2, 32, dtype, scale_q=1.0)
    q = (q.float() * 40).to(dtype)
    check(q, k, v, g, q_off, k_off, causal=False)


@pytest.mark.gpu
def test_scale_and_offset_types():
    from fastmd_amd.ops.attention import segment_attention

    q, k, v, g, q_off, k_off = make([70, 20], [33, 50], 2, 2, 32, torch.float32)
    check(q, k, v, g, q_off, k_off, causal=False, scale=0.7)
    a = [x.cuda() for x in (q, k, v)]
    want = segment_attention(*a, q_off.cuda(), k_off.cuda())
    assert torch.equal(segment_attention(*a, q_off.int().cuda(), k_off.int().cuda()), want)


@pytest.mark.gpu
def test_nothing_to_do():
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    for tq, tk, off in ((0, 0, [0]), (0, 5, [0, 0]), (5, 0, [0, 0]), (4, 4, [0])):
        q, k = torch.ones(tq, 2, 16, device="cuda"), torch.ones(tk, 2, 16, device="cuda")
        o = torch.tensor(off, device="cuda")
        out, saved = segment_attention_forward(q, k, k, o)
        grads = segment_attention_vjp(q, q, k, k, out, saved, o)
        for x in (out, *grads):
            assert not x.any()


@pytest.mark.gpu
def test_offsets_outside_the_buffers_stay_in_bounds():
    """Offsets past the buffers are clamped (an overflowed list's counts), descending ones give empty segments."""
    from fastmd_amd.ops.attention import segment_attention

    q = torch.randn(40, 2, 16, device="cuda")
    out = segment_attention(q, q, q, torch.tensor([0, 30, 4000], device="cuda"))
    want = segment_attention(q, q, q, torch.tensor([0, 30, 40], device="cuda"))
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_other_stream(dtype):
    from fastmd_amd.ops.attention import segment_attention

    q, k, v, g, q_off, k_off = (x.cuda() for x in make([135, 900], [135, 900], 4, 4, 64, dtype))
    want = segment_attention(q, k, v, q_off, k_off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = segment_attention(q * 1, k * 1, v * 1, q_off, k_off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,dtype,causal", [([135], torch.float32, False), ([900, 1, 700], torch.bfloat16, True),
                                                  ([1500, 1300], torch.float32, False)])
def test_captured_and_replayed(lengths, dtype, causal):
    """Forward and VJP in a graph: every replay on new values equals the eager call, which runs between the replays."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    def run(q, k, v, g, off):
        out, saved = segment_attention_forward(q, k, v, off, causal=causal)
        return (out, *segment_attention_vjp(g, q, k, v, out, saved, off, causal=causal))

    held = [x.cuda() for x in make(lengths, lengths, 4, 2, 64, dtype)[:5]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*held)
    for seed in range(1, 5):
        new = [x.cuda() for x in make(lengths, lengths, 4, 2, 64, dtype, seed=seed)[:5]]
        for x, y in zip(held, new):
            x.copy_(y)
        graph.replay()
        want = run(*new)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), seed


@pytest.mark.gpu
def test_rows_past_32_bits():
    """A cache of more than 2^31 elements, segments at both ends, nothing but their rows written."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    q, k, v, g, q_off, k_off = make([3, 5], [70, 300], 8, 4, 128, torch.bfloat16)
    rows = 2 ** 31 // 512 + 5000
    r = oracle.segment_attention(q, k, v, q_off, k_off, causal=True, gout=g)
    b = bounds(r, torch.bfloat16)

    def spread(x):
        y = torch.empty(rows, 4, 128, dtype=x.dtype, device="cuda")
        y[:70], y[-300:] = x[:70].cuda(), x[70:].cuda()
        return y

    k, v = spread(k), spread(v)
    q, g, q_off = q.cuda(), g.cuda(), torch.tensor([0, 3, 3, 8], device="cuda")
    k_off = torch.tensor([0, 70, rows - 300, rows], device="cuda")
    out, saved = segment_attention_forward(q, k, v, q_off, k_off, causal=True)
    compare(out, r["out"], b["out"], "out")
    gq, gk, gv = segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off, causal=True)
    compare(gq, r["gq"], b["gq"], "gq")
    for x, name in ((gk, "gk"), (gv, "gv")):
        compare(torch.cat((x[:70], x[-300:])), r[name], b[name], name)
        assert not any(bool(part.any()) for part in x[70:-300].split(1 << 20))


@pytest.mark.gpu
def test_refusals():
    from fastmd_amd.ops.attention import AttentionSaved, segment_attention, segment_attention_vjp

    row = torch.zeros(4, 6, device="cuda")
    q = torch.zeros(6, 4, 16, device="cuda")
    k = torch.zeros(6, 2, 16, device="cuda")
    off = torch.tensor([0, 6], device="cuda")
    bad = [
        (lambda: segment_attention(q[0], k, k, off), "rows, heads, dim"),
        (lambda: segment_attention(q.half(), k.half(), k.half(), off), "float32 or bfloat16"),
        (lambda: segment_attention(q, k.bfloat16(), k, off), "float32 or bfloat16"),
        (lambda: segment_attention(q, k, k[:5], off), "one shape"),
        (lambda: segment_attention(q, k[..., :8], k[..., :8], off), "head width"),
        (lambda: segment_attention(q[..., :12], k[..., :12], k[..., :12], off), "multiple of 8"),
        (lambda: segment_attention(*[torch.zeros(6, 2, 136, device="cuda")] * 3, off), "multiple of 8"),
        (lambda: segment_attention(q[:, :3], k, k, off), "multiple of the key heads"),
        (lambda: segment_attention(q, k, k, off.float()), "integer vector"),
        (lambda: segment_attention(q, k, k, off, torch.tensor([0, 3, 6], device="cuda")), "segments"),
        (lambda: segment_attention(q, k, k, off, scale=0.0), "scale"),
        (lambda: segment_attention(q, k, k, off, scale=float("nan")), "scale"),
        (lambda: segment_attention(q, k, k, off.cpu()), "GPU"),
        (lambda: segment_attention_vjp(q[:5], q, k, k, q, AttentionSaved(row, row, None), off), "gout"),
        (lambda: segment_attention_vjp(q, q, k, k, q, AttentionSaved(row, row.T, None), off), "saved"),
        (lambda: segment_attention_vjp(*[x.bfloat16() for x in (q, q, k, k, q)], AttentionSaved(row, row, None), off),
         "residual"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_cpu_tensors_are_refused():
    from fastmd_amd.ops.attention import segment_attention

    x = torch.zeros(3, 1, 8)
    with pytest.raises(ValueError, match="GPU"):
        segment_attention(x, x, x, torch.tensor([0, 3]))


def test_entry_points_refuse_what_no_launch_can_honour():
    from fastmd_amd import _abi

    lib = _abi.load()
    call = lambda **kw: lib.fmd_segment_attention(  # noqa: E731
        0, 16, 32, 32, 16, 32, 32, 16, 32, 32, 16, 16, kw.get("tq", 4), 4, 1, kw.get("heads", 2), kw.get("kv", 2),
        kw.get("dim", 16), 0, kw.get("scale", 1.0), kw.get("splits", 1), 16, None, None, None, None, None)
    assert call(heads=3) == 10001 and call(tq=-1) == 10001 and call(scale=0.0) == 10001 and call(splits=2) == 10001
    assert call(dim=136) == 10002 and call(dim=12) == 10002


def test_oracle_closed_forms():
    """Equal scores average the values; one key copies its value; a causal row sees its prefix only."""
    v = torch.arange(12.0).reshape(4, 1, 3).double()
    zero = torch.zeros(4, 1, 3)
    r = oracle.segment_attention(zero, zero, v, [0, 3, 4], [0, 3, 4])
    assert torch.allclose(r["out"][:3, 0], v[:3, 0].mean(0).expand(3, 3))
    assert torch.equal(r["out"][3], v[3])
    r = oracle.segment_attention(zero, zero, v, [0, 4], [0, 4], causal=True)
    assert torch.allclose(r["out"][1, 0], v[:2, 0].mean(0))
    assert r["lse"][0, 3] == pytest.approx(math.log(4))
