"""(h) The norm over groups of channels with its activation: the HIP kernels against the definition in float64, each value within the
bound of its rounding errors that the oracle carries along (before any run: units and counts there)."""
import pytest
import torch

from oracle import blocks as oracle

TYPES = [torch.float32, torch.bfloat16]


def make(rows, channels, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 5 * rows + channels)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return ((r(rows, channels) * (0.5 + r(channels).abs()) + r(channels)).to(dtype), (1 + 0.3 * r(channels)).to(dtype),
            (0.3 * r(channels)).to(dtype), r(rows, channels).to(dtype))


def check(x, groups, w, b, gy, offsets=None, activation=None, eps=1e-5):
    from fastmd_amd.ops.group_norm import group_norm, group_norm_forward, group_norm_vjp

    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    want = oracle.group_norm(x, groups, w, b, offsets, eps, activation, gy)
    args, kw = (c(x), groups, c(w), c(b)), {"offsets": c(offsets), "activation": activation}
    y = group_norm(*args, eps=eps, **kw)
    oracle.near(y, *want[0], "y")
    y2, saved = group_norm_forward(*args, eps=eps, **kw)
    assert torch.equal(y, y2)
    gx, gw, gb = group_norm_vjp(c(gy), *args, saved, **kw)
    oracle.near(gx, *want[1], "gx")
    assert (gw is None) == (w is None) and (gb is None) == (b is None)
    if w is not None:
        oracle.near(gw, *want[2], "gw")
    if b is not None:
        oracle.near(gb, *want[3], "gb")
    alone = group_norm_vjp(c(gy), *args, saved, need_weights=False, **kw)
    assert alone[1] is None and alone[2] is None and torch.equal(alone[0], gx)
    return y, gx


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,groups", [
    (1, 8, 1), (1, 16, 2), (3, 24, 3), (135, 64, 4), (50, 128, 8), (33, 35, 5), (9, 999, 3), (20, 40, 4), (300, 48, 6), (70, 320, 32),
    (7, 700, 1), (5, 2600, 2), (3, 8192, 1), (2, 4099, 1), (600, 12, 1), (2000, 16, 2), (40, 9, 1), (11, 1025, 1), (4, 33 * 64, 64)])
def test_rows_by_themselves(rows, channels, groups, dtype):
    x, w, b, gy = make(rows, channels, dtype)
    check(x, groups, w, b, gy, activation="silu")


def ragged(lengths, lead=0):
    off = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    off[1:] = torch.tensor(lengths).cumsum(0)
    return off + lead


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,groups", [(8, 1), (6, 2), (128, 8), (128, 32), (320, 32), (24, 3), (35, 7), (640, 4), (2048, 2), (4100, 1),
                                             (3, 1), (999, 3), (1000, 1000), (2600, 1300), (1031, 1), (4099, 1), (1042, 1)])
@pytest.mark.parametrize("lengths", [[5, 0, 17, 33, 9], [300], [0, 0, 700, 1, 64], [2] * 40 + [190]])
def test_segments(channels, groups, lengths, dtype):
    """Empty segments, long ones between short ones, a tile's edge inside a segment, rows before and behind all."""
    lead, spare = 3, 5
    lengths = [max(n, 16) if 0 < n < 16 and channels // groups < 4 else n for n in lengths]  # a variance of a few values only where they are not all there is
    x, w, b, gy = make(sum(lengths) + lead + spare, channels, dtype)
    x[:lead] = float("nan")
    x[x.shape[0] - spare:] = float("inf")
    y, gx = check(x, groups, w, b, gy, ragged(lengths, lead), "silu")
    assert not y[:lead].any() and not y[-spare:].any() and not gx[:lead].any() and not gx[-spare:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,groups", [(8192, 1), (16384, 2), (8191, 1), (3 * 8190, 3)])
def test_segments_of_the_widest_groups(channels, groups, dtype):
    x, w, b, gy = make(12, channels, dtype)
    check(x, groups, w, b, gy, ragged([5, 0, 1, 6]), "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("segments", [1, 3, 40])
def test_long_segments(segments, dtype):
    """Sums joined over many tiles; a mean that is large beside the spread."""
    lengths = [1500 + 977 * (i % 3) for i in range(segments)] if segments > 1 else [50000]
    x, w, b, gy = make(sum(lengths), 32, dtype)
    check(x, 4, w, b, gy, ragged(lengths), "silu")
    if dtype == torch.float32:
        check(x + 100.0, 4, w, b, gy, ragged(lengths))


@pytest.mark.gpu
def test_one_very_long_segment_among_many():
    lengths = [3] * 500 + [120000] + [7] * 500
    x, w, b, gy = make(sum(lengths), 16, torch.bfloat16)
    check(x, 2, w, b, gy, ragged(lengths), "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
def test_activations(activation, dtype):
    x, w, b, gy = make(90, 48, dtype)
    check(x, 4, w, b, gy, activation=activation)
    check(x, 4, w, b, gy, ragged([40, 50]), activation)
    check((x * 5).to(dtype), 4, (w * 20).to(dtype), b, gy, ragged([40, 50]), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_relu(dtype):
    """Away from its step (a weight of 1 and a bias far larger than any norm): the value, or nothing, and its slope."""
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    x, _, _, gy = make(60, 32, dtype)
    w, b = torch.ones(32, dtype=dtype), torch.tensor([50.0, -50.0] * 16, dtype=dtype)
    for offsets in (None, ragged([25, 35])):
        want = oracle.group_norm(x, 4, w, b, offsets, name="relu", gy=gy)
        off = None if offsets is None else offsets.cuda()
        y, saved = group_norm_forward(x.cuda(), 4, w.cuda(), b.cuda(), offsets=off, activation="relu")
        grads = group_norm_vjp(gy.cuda(), x.cuda(), 4, w.cuda(), b.cuda(), saved, offsets=off, activation="relu")
        for got, (value, bound) in zip((y, *grads), want):
            oracle.near(got, value, bound)
        assert not y[:, 1::2].any() and not grads[2][1::2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", ["weight", "bias", "none"])
def test_without_parameters(which, dtype):
    x, w, b, gy = make(70, 40, dtype)
    w, b = w if which == "weight" else None, b if which == "bias" else None
    check(x, 5, w, b, gy)
    check(x, 5, w, b, gy, ragged([30, 40]), "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_constant(dtype):
    """No variance: the norm of eps, nothing but the bias; and a single channel in a group."""
    x, w, b, gy = make(50, 32, dtype)
    x[10:20] = 3.0
    check(x, 4, w, b, gy, eps=1e-3)
    x[:] = -2.0
    y, _ = check(x, 4, w, b, gy, ragged([20, 30]), eps=1e-3)
    assert torch.equal(y, b.cuda().expand(50, 32))
    x, w, b, gy = make(50, 6, dtype)
    y, gx = check(x, 6, w, b, gy)  # every group is one value
    assert torch.equal(y, b.cuda().expand(50, 6)) and not gx.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets", [None, [0, 31, 31, 70]])
def test_strides(dtype, offsets):
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    x, w, b, gy = (t.cuda() for t in make(70, 48, dtype))
    off = None if offsets is None else torch.tensor(offsets, device="cuda")

    def run(x, w, b, gy, off=off):
        y, saved = group_norm_forward(x, 3, w, b, offsets=off, activation="silu")
        return (y, *group_norm_vjp(gy, x, 3, w, b, saved, offsets=off, activation="silu"))

    want = oracle.group_norm(*(t.cpu() if torch.is_tensor(t) else t for t in (x, 3, w, b)), offsets, name="silu", gy=gy.cpu())
    shifted = lambda t, n: torch.empty(t.numel() + n, dtype=dtype, device="cuda")[n:].view(t.shape).copy_(t)  # noqa: E731
    wide = lambda t, n: torch.zeros(t.shape[0], t.shape[1] + 2 * n, dtype=dtype, device="cuda")[:, n:n + t.shape[1]].copy_(t)  # noqa: E731
    every = torch.stack((w, b), 1).contiguous()
    for args in ((x, w, b, gy), (wide(x, 8), w, b, wide(gy, 4)), (wide(x, 1), shifted(w, 1), b, gy), (shifted(x, 1), w, b, shifted(gy, 2)),
                 (x.t().contiguous().t(), every[:, 0], every[:, 1], gy), (x, w, b, gy[:1].expand(70, 48))):
        ref = want if args[3].shape[0] == gy.shape[0] and args[3].stride(0) else oracle.group_norm(
            *(t.cpu() if torch.is_tensor(t) else t for t in (x, 3, w, b)), offsets, name="silu", gy=args[3].cpu())
        for got, (value, bound) in zip(run(*args), ref):
            oracle.near(got, value, bound)
    if off is not None:
        for a, c in zip(run(x, w, b, gy, off.int()), run(x, w, b, gy)):
            assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [None, [0, 12, 30]])
def test_autograd_against_differences(offsets):
    from fastmd_amd.ops.group_norm import group_norm

    x, w, b, gy = make(30, 24, torch.float32)
    off = None if offsets is None else torch.tensor(offsets)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = group_norm(leaves[0], 3, leaves[1], leaves[2], offsets=None if off is None else off.cuda(), activation="silu")
    (y * gy.cuda()).sum().backward()
    gen = torch.Generator().manual_seed(1)
    for n in range(3):
        way = torch.randn((x, w, b)[n].shape, generator=gen).double()
        value = []
        for step in (1e-5, -1e-5):
            t = [v.double() for v in (x, w, b)]
            t[n] = t[n] + step * way
            value.append(float((oracle.group_norm(t[0], 3, t[1], t[2], off, name="silu")[0][0] * gy.double()).sum()))
        got = leaves[n].grad.double().cpu() * way
        assert abs(float(got.sum()) - (value[0] - value[1]) / 2e-5) <= 2e-5 * float(got.abs().sum())


@pytest.mark.gpu
def test_second_derivatives_raise():
    from fastmd_amd.ops.group_norm import group_norm

    x = make(10, 24, torch.float32)[0].cuda().requires_grad_()
    (g,) = torch.autograd.grad(group_norm(x, 3).square().sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="first derivatives"):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_graph_replays_with_other_offsets(dtype):
    """The offsets are read on the device: a captured call follows them."""
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    x, w, b, gy = (t.cuda() for t in make(3000, 64, dtype))
    off = torch.tensor([0, 1000, 2000, 3000], device="cuda")

    def run(x, off):
        y, saved = group_norm_forward(x, 4, w, b, offsets=off, activation="silu")
        return (y, *group_norm_vjp(gy, x, 4, w, b, saved, offsets=off, activation="silu"))

    sx, so = x.clone(), off.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(sx, so)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(sx, so)
    for k, ends in enumerate(([0, 1000, 2000, 3000], [0, 5, 5, 2990], [10, 2900, 2950, 3000], [0, 0, 0, 3000])):
        nx = x * (1 + k)
        now = torch.tensor(ends, device="cuda")
        want = run(nx, now)
        sx.copy_(nx)
        so.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_repeatable(dtype):
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    x, w, b, gy = (t.cuda() for t in make(20000, 64, dtype))
    for off in (None, torch.tensor([0, 9, 8000, 20000], device="cuda")):
        runs = []
        for _ in range(3):
            y, saved = group_norm_forward(x, 4, w, b, offsets=off)
            runs.append((y, *group_norm_vjp(gy, x, 4, w, b, saved, offsets=off)))
        for r in runs[1:]:
            for a, c in zip(r, runs[0]):
                assert torch.equal(a, c)


@pytest.mark.gpu
def test_offsets_that_do_not_ascend_stay_in_the_buffers():
    """Which rows such a call computes is open: nothing outside the buffers is touched, and the next call is right."""
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    x, w, b, gy = (t.cuda() for t in make(700, 64, torch.float32))
    for ends in ([0, 500, 200, 700], [700, 0], [-50, 900, 20], [300, 299, 298, 0, 700]):
        off = torch.tensor(ends, device="cuda")
        _, saved = group_norm_forward(x, 4, w, b, offsets=off)
        group_norm_vjp(gy, x, 4, w, b, saved, offsets=off)
        torch.cuda.synchronize()
    check(*(t.cpu() if torch.is_tensor(t) else t for t in (x, 4, w, b, gy)), ragged([300, 400]))


@pytest.mark.gpu
def test_nothing_to_do():
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    for rows, off in ((0, None), (0, [0, 0, 0]), (9, [0]), (9, [0, 0, 0]), (9, [9, 9])):
        x, w, b, gy = (t.cuda() for t in make(rows, 16, torch.float32))
        offsets = None if off is None else torch.tensor(off, device="cuda")
        y, saved = group_norm_forward(x, 2, w, b, offsets=offsets)
        gx, gw, gb = group_norm_vjp(gy, x, 2, w, b, saved, offsets=offsets)
        assert y.shape == x.shape and not y.any() and not gx.any() and not gw.any() and not gb.any()


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [False, True])
def test_values_past_32_bits(offsets):
    from fastmd_amd.ops.group_norm import group_norm

    rows, n = 2 ** 31 // 512 + 300, 300
    x, w, b, _ = make(n, 512, torch.bfloat16)
    big = torch.zeros(rows, 512, dtype=torch.bfloat16, device="cuda")
    big[-n:] = x.cuda()
    off = torch.tensor([0, rows - n, rows - 100, rows], device="cuda") if offsets else None
    y = group_norm(big, 8, w.cuda(), b.cuda(), offsets=off)
    want = oracle.group_norm(x, 8, w, b, torch.tensor([0, 200, 300]) if offsets else None)[0]
    oracle.near(y[-n:], *want)
    assert torch.equal(y[5], b.cuda())


@pytest.mark.gpu
def test_refusals():
    from fastmd_amd.ops.group_norm import group_norm, group_norm_forward, group_norm_vjp

    x, w, b, gy = (t.cuda() for t in make(10, 24, torch.float32))
    off = torch.tensor([0, 4, 10], device="cuda")
    _, saved = group_norm_forward(x, 3, w, b)
    bad = [
        (lambda: group_norm(x[0], 3), "rows, channels"),
        (lambda: group_norm(x.half(), 3), "float32 or bfloat16"),
        (lambda: group_norm(x, 5), "multiple of the groups"),
        (lambda: group_norm(x, 0), "multiple of the groups"),
        (lambda: group_norm(x, 48), "multiple of the groups"),
        (lambda: group_norm(torch.zeros(2, 8200, device="cuda"), 1), "at most"),
        (lambda: group_norm(torch.zeros(2, 65536, device="cuda"), 65536), "at most 65535 groups"),
        (lambda: group_norm(x, 3, w[:20]), "weight"),
        (lambda: group_norm(x, 3, w, b.bfloat16()), "bias"),
        (lambda: group_norm(x, 3, offsets=off.float()), "offsets"),
        (lambda: group_norm(x, 3, offsets=off[None]), "offsets"),
        (lambda: group_norm(x, 3, offsets=off.cpu()), "GPU"),
        (lambda: group_norm(x, 3, eps=-1.0), "eps"),
        (lambda: group_norm(x, 3, eps=float("nan")), "eps"),
        (lambda: group_norm(x, 3, activation="tanh"), "activation"),
        (lambda: group_norm_vjp(gy[:5], x, 3, w, b, saved), "gy"),
        (lambda: group_norm_vjp(gy, x, 3, w, b, saved, offsets=off), "saved"),
        (lambda: group_norm_vjp(gy, x, 6, w, b, saved), "saved"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_cpu_tensors_are_refused():
    from fastmd_amd.ops.group_norm import group_norm

    with pytest.raises(ValueError, match="GPU"):
        group_norm(torch.zeros(2, 8), 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets", [[0, 300, 100, 400], [400, 0, 400], [399, -5, 700, 2, 400], [400, 300, 200, 0], [0, 9000, 40, 9000]])
def test_descending_offsets_stay_in_bounds(offsets, dtype):
    """Such a call ends, and the inputs keep their values (which rows it computes is open)."""
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    rows = max(max(offsets) - 300 if 700 in offsets else max(offsets), 400)
    x, w, b, gy = (t.cuda() for t in make(rows, 32, dtype))
    kept = [t.clone() for t in (x, w, b, gy)]
    off = torch.tensor(offsets, device="cuda")
    for groups in (1, 32):
        _, saved = group_norm_forward(x, groups, w, b, offsets=off)
        group_norm_vjp(gy, x, groups, w, b, saved, offsets=off)
    torch.cuda.synchronize()
    for a, k in zip((x, w, b, gy), kept):
        assert torch.equal(a, k)
