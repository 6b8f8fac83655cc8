"""(h) The gated feed-forward block: the HIP kernels against the definition in float64, each value within the bound of its rounding
errors that the oracle carries along (before any run: units and counts there)."""
import pytest
import torch

from oracle import blocks as oracle

TYPES = [torch.float32, torch.bfloat16]


def make(rows, width, hidden, out, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * rows + 3 * width + hidden)
    r = lambda *s, f=1.0: (torch.randn(*s, generator=g) * f).to(dtype)  # noqa: E731
    return (r(rows, width), r(hidden, width, f=width ** -0.5), r(hidden, width, f=width ** -0.5), r(out, hidden, f=hidden ** -0.5),
            r(rows, out))


def check(x, wg, wu, wd, gy, activation="silu"):
    from fastmd_amd.ops.feed_forward import gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp

    args = [t.cuda() for t in (x, wg, wu, wd)]
    want = oracle.gated(x, wg, wu, wd, activation, gy)
    y = gated_feed_forward(*args, activation=activation)
    oracle.near(y, *want[0], "y")
    y2, saved = gated_feed_forward_forward(*args, activation=activation)
    oracle.near(y2, *want[0], "y of the forward")
    g = gy.cuda()
    both = gated_feed_forward_vjp(g, *args, saved, activation=activation)
    for name, got, (value, bound) in zip(("gx", "g_gate", "g_up", "g_down"), both, want[1:]):
        assert got.dtype == x.dtype
        oracle.near(got, value, bound, name)
    alone = gated_feed_forward_vjp(g, *args, saved, activation=activation, need_weights=False)
    assert alone[1:] == (None, None, None)
    oracle.near(alone[0], *want[1], "gx alone")
    weights = gated_feed_forward_vjp(g, *args, saved, activation=activation, need_x=False)
    assert weights[0] is None
    for got, (value, bound) in zip(weights[1:], want[2:]):
        oracle.near(got, value, bound, "weights alone")
    return y, both


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,hidden,out", [
    (1, 1, 1, 1), (1, 8, 8, 8), (2, 16, 24, 16), (5, 7, 13, 3), (16, 64, 128, 64), (17, 40, 100, 40), (31, 128, 344, 128), (32, 72, 96, 72),
    (33, 96, 200, 64), (64, 64, 64, 64), (65, 33, 67, 34), (135, 64, 128, 64), (129, 130, 257, 131), (300, 256, 680, 256),
    (1, 512, 1376, 512), (8, 520, 1100, 264), (700, 24, 40, 24), (257, 264, 136, 520)])
def test_sizes(rows, width, hidden, out, dtype):
    check(*make(rows, width, hidden, out, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
@pytest.mark.parametrize("rows,width,hidden", [(9, 24, 40), (150, 64, 128), (140, 200, 300)])
def test_activations(rows, width, hidden, activation, dtype):
    check(*make(rows, width, hidden, width, dtype), activation=activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,hidden", [(9, 24, 40), (150, 64, 128), (140, 200, 300)])
def test_relu_on_whole_numbers(rows, width, hidden, dtype):
    """Every product and sum is exact in float32, so which side of 0 a value is on is no matter of rounding: many are 0,
    where the slope is 0."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    g = torch.Generator().manual_seed(rows)
    r = lambda *s: torch.randint(-1, 2, s, generator=g).to(dtype)  # noqa: E731
    x, wg, wu, wd, gy = r(rows, width), r(hidden, width), r(hidden, width), r(width, hidden), r(rows, width)
    args = [t.cuda() for t in (x, wg, wu, wd)]
    want = oracle.gated(x, wg, wu, wd, "relu", gy)
    assert bool(((x.double() @ wg.double().T) == 0).any())
    y, saved = gated_feed_forward_forward(*args, activation="relu")
    for got, (value, bound) in zip((y, *gated_feed_forward_vjp(gy.cuda(), *args, saved, activation="relu")), want):
        oracle.near(got, value, bound)
        if dtype == torch.float32:
            assert torch.equal(got.double().cpu(), value)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 40, 150])
def test_strides(dtype, rows):
    """Columns of wider buffers, transposed weights, rows off 16 bytes, a packed pair of projections: the same values."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(rows, 48, 80, 48, dtype))

    def run(x, wg, wu, wd, gy):
        y, saved = gated_feed_forward_forward(x, wg, wu, wd)
        return (y, *gated_feed_forward_vjp(gy, x, wg, wu, wd, saved))

    want = run(x, wg, wu, wd, gy)
    off = lambda t: torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    wide = lambda t, n: torch.zeros(t.shape[0], t.shape[1] + n, dtype=dtype, device="cuda")[:, n // 2:n // 2 + t.shape[1]].copy_(t)  # noqa: E731
    turned = lambda t: t.t().contiguous().t()  # noqa: E731
    packed = torch.cat((wg, wu))
    for args in ((wide(x, 16), packed[:80], packed[80:], wd, wide(gy, 32)), (wide(x, 6), off(wg), wu, wide(wd, 2), off(gy)),
                 (turned(x), turned(wg), wide(wu, 8), turned(wd), turned(gy)), (off(x), wg, off(wu), off(wd), gy)):
        for a, b in zip(run(*args), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_do_not_reach_each_other(dtype):
    """A row that is not finite makes its own results NaN, and no other row's; what lies behind the rows in memory is not used."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp

    for rows, width, hidden in ((20, 24, 40), (300, 64, 136), (200, 136, 272)):
        x, wg, wu, wd, gy = (t.cuda() for t in make(rows, width, hidden, width, dtype))
        want = gated_feed_forward(x, wg, wu, wd)
        big = torch.full((rows + 9, width + 8), float("nan"), dtype=dtype, device="cuda")
        big[:rows, :width] = x
        bad = big[:rows, :width]
        assert torch.equal(gated_feed_forward(bad, wg, wu, wd), want)
        bad[3, 5] = float("nan")
        bad[7, 0] = float("inf")
        got, saved = gated_feed_forward_forward(bad, wg, wu, wd)
        gx = gated_feed_forward_vjp(gy, bad, wg, wu, wd, saved, need_weights=False)[0]
        keep = [i for i in range(rows) if i not in (3, 7)]
        assert torch.isnan(got[3]).all() and not torch.isfinite(got[7]).any()
        assert torch.equal(got[keep], want[keep]) and torch.isfinite(gx[keep]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_values(dtype):
    """Gates far from 0 on both sides: the activation is 0 or the value, the slope 0 or 1."""
    x, wg, wu, wd, gy = make(50, 16, 24, 16, dtype)
    check((x * 300).to(dtype), wg, wu, wd, gy)
    check((x * 300).to(dtype), wg, wu, wd, gy, activation="gelu")
    check((x * 1e-3).to(dtype), wg, wu, wd, gy)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 200])
def test_autograd_against_differences(rows):
    from fastmd_amd.ops.feed_forward import gated_feed_forward

    leaves = make(rows, 24, 40, 16, torch.float32, seed=3)
    gy = leaves[4]
    on = [t.cuda().requires_grad_() for t in leaves[:4]]
    (gated_feed_forward(*on) * gy.cuda()).sum().backward()
    gen = torch.Generator().manual_seed(1)
    for n in range(4):
        way = torch.randn(leaves[n].shape, generator=gen).double()
        value = []
        for step in (1e-5, -1e-5):
            t = [v.double() for v in leaves[:4]]
            t[n] = t[n] + step * way
            a, _ = oracle.act(t[0] @ t[1].T, "silu")
            value.append(float((((a * (t[0] @ t[2].T)) @ t[3].T) * gy.double()).sum()))
        got = on[n].grad.double().cpu() * way
        assert abs(float(got.sum()) - (value[0] - value[1]) / 2e-5) <= 1e-5 * float(got.abs().sum())


@pytest.mark.gpu
def test_autograd_by_need():
    """Leaves that need no gradient get none; a gradient that is a broadcast view."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward

    x, wg, wu, wd, _ = (t.cuda() for t in make(40, 24, 40, 16, torch.float32))
    a = x.clone().requires_grad_()
    gated_feed_forward(a, wg, wu, wd).sum().backward()
    w = [t.clone().requires_grad_() for t in (wg, wu, wd)]
    gated_feed_forward(x, *w).sum().backward()
    want = oracle.gated(*(t.cpu() for t in (x, wg, wu, wd)), "silu", torch.ones(40, 16))
    for got, (value, bound) in zip((a.grad, *(t.grad for t in w)), want[1:]):
        oracle.near(got, value, bound)
    half = [t.clone() for t in (wg, wu, wd)]
    half[2].requires_grad_()
    gated_feed_forward(x, *half).sum().backward()
    assert half[0].grad is None and torch.equal(half[2].grad, w[2].grad)


@pytest.mark.gpu
def test_shared_weights_add_their_gradients():
    from fastmd_amd.ops.feed_forward import gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp

    x, w, _, wd, gy = (t.cuda() for t in make(40, 24, 40, 24, torch.float32))
    leaf = w.clone().requires_grad_()
    gated_feed_forward(x, leaf, leaf, wd).backward(gy)
    _, saved = gated_feed_forward_forward(x, w, w, wd)
    _, a, b, _ = gated_feed_forward_vjp(gy, x, w, w, wd, saved)
    assert torch.equal(leaf.grad, a + b)


@pytest.mark.gpu
def test_second_derivatives_and_tangents_raise():
    from torch.autograd import forward_ad

    from fastmd_amd.ops.feed_forward import gated_feed_forward

    x, wg, wu, wd, _ = (t.cuda() for t in make(10, 24, 40, 24, torch.float32))
    x.requires_grad_()
    (g,) = torch.autograd.grad(gated_feed_forward(x, wg, wu, wd).sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="first derivatives"):
        g.sum().backward()
    with forward_ad.dual_level(), pytest.raises(Exception):
        gated_feed_forward(forward_ad.make_dual(x.detach(), torch.ones_like(x)), wg, wu, wd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,hidden", [(3, 64, 128), (200, 64, 128), (300, 256, 680), (4000, 136, 264)])
def test_repeatable(rows, width, hidden, dtype):
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(rows, width, hidden, width, dtype))

    def run():
        y, saved = gated_feed_forward_forward(x, wg, wu, wd)
        return (y, *gated_feed_forward_vjp(gy, x, wg, wu, wd, saved))

    first = run()
    for _ in range(3):
        for a, b in zip(run(), first):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 300])
def test_graph_replays(dtype, rows):
    """Captured with its VJP and replayed on other inputs, with eager calls between the replays."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(rows, 136, 200, 136, dtype))

    def run(x, gy):
        y, saved = gated_feed_forward_forward(x, wg, wu, wd)
        return (y, *gated_feed_forward_vjp(gy, x, wg, wu, wd, saved))

    sx, sg = x.clone(), gy.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(sx, sg)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(sx, sg)
    for k in range(4):
        nx, ng = x * (1 + k), gy.flip(0) if k % 2 else gy
        want = run(nx, ng)
        sx.copy_(nx)
        sg.copy_(ng)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_on_another_stream():
    from fastmd_amd.ops.feed_forward import gated_feed_forward

    x, wg, wu, wd, _ = (t.cuda() for t in make(500, 136, 200, 136, torch.bfloat16))
    want = gated_feed_forward(x, wg, wu, wd)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(gated_feed_forward(x, wg, wu, wd))
    torch.cuda.synchronize()
    for y in outs:
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_no_rows():
    from fastmd_amd.ops.feed_forward import gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(0, 24, 40, 16, torch.bfloat16))
    assert gated_feed_forward(x, wg, wu, wd).shape == (0, 16)
    _, saved = gated_feed_forward_forward(x, wg, wu, wd)
    gx, *gw = gated_feed_forward_vjp(gy, x, wg, wu, wd, saved)
    assert gx.shape == (0, 24) and not any(bool(t.any()) for t in gw) and [t.shape for t in gw] == [wg.shape, wu.shape, wd.shape]


@pytest.mark.gpu
def test_values_past_32_bits():
    """More than 2^31 values in x, in what is saved, and in y; a few rows checked."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward

    rows, width = 2 ** 31 // 2048 + 300, 2048
    x, wg, wu, wd, _ = make(300, width, 16, width, torch.bfloat16)
    big = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    big[-300:] = x.cuda()
    y = gated_feed_forward(big, wg.cuda(), wu.cuda(), wd.cuda())
    oracle.near(y[-300:], *oracle.gated(x, wg, wu, wd, "silu")[0])
    assert not y[:-300].any()


@pytest.mark.gpu
def test_refusals():
    from fastmd_amd.ops.feed_forward import gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(5, 24, 40, 16, torch.float32))
    _, saved = gated_feed_forward_forward(x, wg, wu, wd)
    bad = [
        (lambda: gated_feed_forward(x[0], wg, wu, wd), "matrix"),
        (lambda: gated_feed_forward(x.half(), wg.half(), wu.half(), wd.half()), "float32 or bfloat16"),
        (lambda: gated_feed_forward(x, wg.bfloat16(), wu, wd), "float32 or bfloat16"),
        (lambda: gated_feed_forward(x[:, :23], wg, wu, wd), "fit together"),
        (lambda: gated_feed_forward(x, wg, wu[:39], wd), "fit together"),
        (lambda: gated_feed_forward(x, wg, wu, wd[:, :39]), "fit together"),
        (lambda: gated_feed_forward(x[:, :0], wg[:, :0], wu[:, :0], wd), "from 1"),
        (lambda: gated_feed_forward(x, wg[:0], wu[:0], wd[:, :0]), "from 1"),
        (lambda: gated_feed_forward(x, wg, wu, wd, activation="tanh"), "activation"),
        (lambda: gated_feed_forward(x[:1].expand(2 ** 29, 24), wg, wu, wd), "fewer than 2\\^29 rows"),
        (lambda: gated_feed_forward_vjp(gy[:, :8], x, wg, wu, wd, saved), "gy"),
        (lambda: gated_feed_forward_vjp(gy.bfloat16(), x, wg, wu, wd, saved), "gy"),
        (lambda: gated_feed_forward_vjp(gy, x[:4], wg, wu, wd, saved), "gy"),
        (lambda: gated_feed_forward(x.cpu(), wg, wu, wd), "GPU"),
        (lambda: gated_feed_forward(x, wg, wu, wd.cpu()), "GPU"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_cpu_tensors_are_refused():
    from fastmd_amd.ops.feed_forward import gated_feed_forward

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="GPU"):
        gated_feed_forward(x, torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))


def test_entry_points_refuse_more_tiles_than_a_launch_takes():
    """Before anything is launched: the operands' layouts would go to a workspace that is not there."""
    from fastmd_amd import _abi

    lib = _abi.load()
    rows, width, hidden, out = 2 ** 31 - 1, 64, 2048, 64
    for bf16 in (0, 1):
        assert lib.fmd_gated_ffn(bf16, 1, 15, 16, width, 16, 16, width, 16, hidden, rows, width, hidden, out, 16, None, None, None,
                                 None) == 10001
        assert lib.fmd_gated_ffn_bwd(bf16, 1, 15, 16, width, 16, 16, width, 16, hidden, rows, width, hidden, out, 16, out, 16, 16,
                                     16, 16, 16, 16, None, None) == 10001
