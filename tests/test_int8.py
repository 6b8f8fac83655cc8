"""(h) Rows and products in 8-bit integers: integers equal to the definition's, results within three float32 roundings (the sum's,
two products, and a bias' sum) and the one of the result's type."""
import pytest
import torch

from oracle import blocks as oracle

TYPES = [torch.float32, torch.bfloat16]


def make(rows, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 3 * rows + width)
    return (torch.randn(rows, width, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 16), (5, 17), (300, 64), (9, 512), (7, 520), (6, 1024), (5, 2048), (4, 4100), (3, 8192),
                                        (2, 9000), (2, 30001)])
def test_rows(rows, width, dtype):
    from fastmd_amd.ops.int8 import quantize_rows

    x = make(rows, width, dtype)
    if rows > 2:
        x[1] = 0.0
        x[2, 0] = x[2].abs().max() * 2  # a power of two times the others: many ties
        x[0] = x[0].sign() * 2.0
    q = quantize_rows(x.cuda())
    want, scale = oracle.quantize(x)
    assert q.values.shape == x.shape and torch.equal(q.values.cpu().double(), want) and torch.equal(q.scales.cpu(), scale)
    assert torch.equal(q.dense().cpu(), want.float() * scale[:, None])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,out", [(1, 1, 1), (1, 16, 16), (3, 17, 5), (16, 512, 300), (17, 100, 77), (32, 1030, 64), (33, 256, 129), (135, 100, 77),
                                            (300, 256, 512), (1000, 4097, 130), (64, 64, 64), (1, 4096, 1000), (500, 2050, 700)])
def test_products(rows, width, out, dtype):
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows

    x, w = make(rows, width, dtype), make(out, width, torch.float32, seed=1)
    q, scale = oracle.quantize(x)
    qw, w_scale = oracle.quantize(w)
    weight = quantize_rows(w.cuda())
    y = linear_int8(x.cuda(), weight)
    assert y.dtype == dtype
    oracle.near(y, *oracle.linear_int8(q, scale, qw, w_scale, None, dtype))
    bias = torch.randn(out, generator=torch.Generator().manual_seed(2))
    for kind in TYPES:
        y = linear_int8(quantize_rows(x.cuda()), weight, bias.cuda(), dtype=kind)
        oracle.near(y, *oracle.linear_int8(q, scale, qw, w_scale, bias, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [131071, 70000])
def test_the_largest_sums(width):
    """All products 127^2 (and all -127^2): the sums stay within 32 bits and are exact."""
    from fastmd_amd.ops.int8 import Int8Rows, linear_int8

    one = torch.ones(3, device="cuda")
    for sign in (1, -1):
        a = Int8Rows(torch.full((3, width), 127, dtype=torch.int8, device="cuda"), one)
        b = Int8Rows(torch.full((3, width), 127 * sign, dtype=torch.int8, device="cuda"), one)
        assert torch.equal(linear_int8(a, b), torch.full((3, 3), float(sign * 127 * 127 * width), device="cuda"))


@pytest.mark.gpu
def test_strides_and_what_lies_past_the_width():
    from fastmd_amd.ops.int8 import Int8Rows, linear_int8, quantize_rows

    x, w = make(40, 100, torch.float32), make(60, 100, torch.float32, seed=1)
    want = linear_int8(x.cuda(), quantize_rows(w.cuda()))
    wide = torch.full((40, 131), float("nan"), device="cuda")
    wide[:, 7:107] = x.cuda()
    assert torch.equal(linear_int8(wide[:, 7:107], quantize_rows(w.cuda())), want)
    assert torch.equal(linear_int8(x.t().contiguous().cuda().t(), quantize_rows(w.cuda())), want)
    q, qw = quantize_rows(x.cuda()), quantize_rows(w.cuda())
    for n, ld in ((0, 100), (0, 128), (16, 160), (3, 112), (1, 101)):
        def within(v):
            t = torch.full((v.shape[0], ld + n), 77, dtype=torch.int8, device="cuda")
            t[:, n:n + 100] = v
            return t[:, n:n + 100]
        got = linear_int8(Int8Rows(within(q.values), q.scales), Int8Rows(within(qw.values), qw.scales))
        assert torch.equal(got, want)
    scales = torch.stack((qw.scales, qw.scales), 1)[:, 0]
    assert torch.equal(linear_int8(q, Int8Rows(qw.values.t().contiguous().t(), scales)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_not_finite(dtype):
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows

    x, w = make(40, 64, dtype).cuda(), quantize_rows(make(50, 64, torch.float32, seed=1).cuda())
    want = linear_int8(x, w)
    x[3, 5], x[7, 0], x[9, 1] = float("nan"), float("inf"), -float("inf")
    got = linear_int8(x, w)
    keep = [i for i in range(40) if i not in (3, 7, 9)]
    assert torch.isnan(got[[3, 7, 9]]).all() and torch.equal(got[keep], want[keep])


@pytest.mark.gpu
def test_graph_replays():
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows

    x, w = make(40, 640, torch.bfloat16).cuda(), quantize_rows(make(500, 640, torch.float32, seed=1).cuda())
    static = x.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        linear_int8(static, w)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_int8(static, w)
    for k in range(4):
        want = linear_int8(x * (k + 1), w)
        static.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_values_past_32_bits():
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows

    rows, width = 2 ** 31 // 4096 + 200, 4096
    x, w = make(200, width, torch.bfloat16), make(8, width, torch.float32, seed=1)
    big = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    big[-200:] = x.cuda()
    y = linear_int8(big, quantize_rows(w.cuda()))
    oracle.near(y[-200:], *oracle.linear_int8(*oracle.quantize(x), *oracle.quantize(w), None, torch.bfloat16))
    assert not y[:-200].any()


@pytest.mark.gpu
def test_nothing_to_do_and_refusals():
    from fastmd_amd.ops.int8 import Int8Rows, linear_int8, quantize_rows

    x, w = make(5, 32, torch.float32).cuda(), quantize_rows(make(6, 32, torch.float32, seed=1).cuda())
    assert linear_int8(x[:0], w).shape == (0, 6) and quantize_rows(x[:0]).values.shape == (0, 32)
    bad = [
        (lambda: quantize_rows(x[0]), "matrix"),
        (lambda: quantize_rows(x.half()), "float32 or bfloat16"),
        (lambda: quantize_rows(x[:, :0]), "one column"),
        (lambda: quantize_rows(x.clone().requires_grad_()), "no gradient"),
        (lambda: quantize_rows(x.cpu()), "GPU"),
        (lambda: linear_int8(x, w.values), "Int8Rows"),
        (lambda: linear_int8(x.clone().requires_grad_(), w), "no gradient"),
        (lambda: linear_int8(x[:, :31], w), "one width"),
        (lambda: linear_int8(x[:1].expand(2 ** 29, 32), w), "fewer than 2\\^29 rows"),
        (lambda: linear_int8(x, Int8Rows(w.values.short(), w.scales)), "weight must be int8"),
        (lambda: linear_int8(x, Int8Rows(w.values, w.scales[:5])), "weight must be int8"),
        (lambda: linear_int8(x, Int8Rows(w.values, w.scales.double())), "weight must be int8"),
        (lambda: linear_int8(x, w, torch.zeros(5, device="cuda")), "bias"),
        (lambda: linear_int8(x, w, dtype=torch.float16), "result"),
        (lambda: linear_int8(x, Int8Rows(w.values.cpu(), w.scales)), "GPU"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_cpu_tensors_are_refused():
    from fastmd_amd.ops.int8 import quantize_rows

    with pytest.raises(ValueError, match="GPU"):
        quantize_rows(torch.zeros(2, 8))


def test_entry_points_refuse_what_no_launch_can_honour():
    from fastmd_amd import _abi

    lib = _abi.load()
    linear = lambda rows=4, width=32, out=8, x_ld=32, w=16: lib.fmd_linear_int8(  # noqa: E731
        0, 16, x_ld, 16, w, 32, 16, None, rows, width, out, 16, 16, None)
    assert linear(rows=0) == 10001 and linear(width=131072) == 10001 and linear(x_ld=31) == 10001 and linear(w=8) == 10001
    assert lib.fmd_quantize_rows(0, 16, 32, 4, 32, 16, 31, 16, None) == 10001
    norm = lambda **k: lib.fmd_group_norm(0, k.get("act", 0), 16, 24, None, None, k.get("rows", 4), k.get("channels", 24),  # noqa: E731
                                          k.get("groups", 3), k.get("off"), 2, k.get("eps", 1e-5), 16, None, None, None, None)
    assert norm(groups=5) == 10001 and norm(rows=0) == 10001 and norm(act=4) == 10001 and norm(eps=-1.0) == 10001
    assert norm(channels=24600) == 10001 and norm(off=16) == 10001
    ffn = lambda **k: lib.fmd_gated_ffn(1, k.get("act", 1), 0, k.get("x", 16), k.get("ld", 32), 16, 16, k.get("gate", 32), 16, 40,  # noqa: E731
                                        k.get("rows", 4), 32, k.get("hidden", 40), 8, 16, None, None, 16, None)
    assert ffn(rows=0) == 10001 and ffn(act=9) == 10001 and ffn(x=8) == 10001 and ffn(ld=33) == 10001 and ffn(hidden=36) == 10001
    assert ffn(gate=36) == 10001
