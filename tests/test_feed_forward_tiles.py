"""(h) The gated feed-forward block's forms for larger calls against the definition in float64: tiles in LDS (every shape and split, laid
out operands, odd widths) and products straight from memory with every number of rows a wave. Each list says which form a size
takes, and a host test holds it to that."""
import pytest
import torch

from feed_forward_forms import forms
from oracle import blocks as oracle
from test_feed_forward import check, make
from test_host_math import run_host

F32, BF16 = torch.float32, torch.bfloat16

TILES = [
    (F32, 1500, 301, 1003, 299),   # odd widths
    (F32, 700, 520, 1376, 264),    # K shared
    (F32, 5000, 96, 1100, 40),     # narrow results
    (F32, 9000, 40, 1032, 130),
    (F32, 16384, 136, 520, 256),   # K not shared, in the VJP for x
    (F32, 16875, 256, 680, 256),
    (F32, 6000, 520, 1032, 264),
    (F32, 131, 1300, 2100, 1290),  # few rows, large weights
    (BF16, 1500, 301, 1003, 299),
    (BF16, 700, 520, 1376, 264),
    (BF16, 3000, 96, 1100, 40),
    (BF16, 8200, 33, 520, 130),
    (BF16, 40000, 40, 300, 40),    # K not shared
    (BF16, 9000, 520, 1376, 1032),
    (BF16, 5000, 1100, 1000, 520),
    (BF16, 131, 1000, 2100, 990),
    (BF16, 600, 344, 872, 344),    # whole vectors: nothing is laid out
]
# 1 024 tiles of 256 rows by 128 columns of the hidden layer and more; narrow inputs keep the oracle quick
ONE = [(F32, 8200, 64, 120, 64), (F32, 8300, 40, 100, 33), (BF16, 8200, 64, 120, 64), (BF16, 9000, 17, 90, 23)]  # 32 rows of a workgroup
MANY = [(F32, 8200, 16, 4100, 24), (BF16, 8200, 16, 4100, 24)]


def is_bf16(dtype):
    return int(dtype == BF16)


def partial(dtype, rows, width, hidden, out):
    """Bytes of the sums of split tiles, in the VJP for x and in that for all."""
    from fastmd_amd import _abi

    lib, bf16 = _abi.load(), is_bf16(dtype)
    up = lambda x, n: -(-x // n) * n  # noqa: E731
    planes, kept = (1, 2) if bf16 else (3, 3)
    lay = lambda rows, cols: up(rows * up(cols, 8) * 2 * planes, 256)  # noqa: E731
    weights, gradients = 2 * lay(hidden, width) + lay(out, hidden), up(2 * rows * up(hidden, 8) * 2 * kept, 256)
    size = lib.fmd_gated_ffn_bwd_work_size
    return (size(bf16, rows, width, hidden, out, 15, 1, 0) - weights - lay(rows, out) - gradients,
            size(bf16, rows, width, hidden, out, 15, 1, 1) - weights - lay(rows, out) - gradients - lay(rows, width))


def test_the_sizes_take_tiles():
    for dtype, *size in TILES + MANY:
        assert forms(is_bf16(dtype), *size) == ("tiles", "tiles"), size
    for dtype, *size in ONE:
        assert forms(is_bf16(dtype), *size) == ("one", "one") and size[0] >= 32 * 256, size
    for _, rows, _, hidden, _ in MANY:
        assert -(-rows // 256) * -(-hidden // 128) >= 1024
    sums = [partial(dtype, *size) for dtype, *size in TILES]
    assert all(x >= 0 and a >= 0 for x, a in sums)
    for bf16 in (0, 1):  # K shared and not, in the VJP of either type
        split = [x > 0 for (x, _), (dtype, *_) in zip(sums, TILES) if is_bf16(dtype) == bf16]
        assert any(split) and not all(split)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,hidden,out", ONE)
def test_one_kernel_over_many_rows(dtype, rows, width, hidden, out):
    check(*make(rows, width, hidden, out, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,hidden,out", TILES + MANY)
def test_tiles(dtype, rows, width, hidden, out):
    check(*make(rows, width, hidden, out, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_activations_in_tiles(dtype, activation):
    check(*make(700, 520, 1376, 264, dtype), activation=activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,hidden,out", [size for size in TILES if size[1] in (131, 600, 700)])
def test_strides_in_tiles(dtype, rows, width, hidden, out):
    """Columns of wider buffers, transposed weights, rows off 16 bytes, a packed pair of projections: the same values, whatever lies
    beside them."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(rows, width, hidden, out, dtype))

    def run(x, wg, wu, wd, gy):
        y, saved = gated_feed_forward_forward(x, wg, wu, wd)
        return (y, *gated_feed_forward_vjp(gy, x, wg, wu, wd, saved))

    want = run(x, wg, wu, wd, gy)
    off = lambda t: torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731

    def wide(t, n):
        buffer = torch.full((t.shape[0], t.shape[1] + n), float("nan"), dtype=dtype, device="cuda")
        return buffer[:, n // 2:n // 2 + t.shape[1]].copy_(t)

    turned = lambda t: t.t().contiguous().t()  # noqa: E731
    packed = torch.cat((wg, wu))
    for args in ((wide(x, 16), packed[:hidden], packed[hidden:], wd, wide(gy, 32)), (wide(x, 6), off(wg), wu, wide(wd, 2), off(gy)),
                 (turned(x), turned(wg), wide(wu, 8), turned(wd), turned(gy)), (off(x), wg, off(wu), off(wd), gy)):
        for a, b in zip(run(*args), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_that_is_not_finite_in_tiles(dtype):
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = (t.cuda() for t in make(700, 520, 1376, 264, dtype))
    y, saved = gated_feed_forward_forward(x, wg, wu, wd)
    gx = gated_feed_forward_vjp(gy, x, wg, wu, wd, saved, need_weights=False)[0]
    x[300, 519], gy[10, 0] = float("nan"), float("inf")
    got, saved = gated_feed_forward_forward(x, wg, wu, wd)
    got_x = gated_feed_forward_vjp(gy, x, wg, wu, wd, saved, need_weights=False)[0]
    keep = torch.tensor([i for i in range(700) if i not in (10, 300)], device="cuda")
    assert torch.isnan(got[300]).all() and torch.isnan(got_x[300]).all() and not torch.isfinite(got_x[10]).any()
    assert torch.equal(got[keep], y[keep]) and torch.equal(got[10], y[10]) and torch.equal(got_x[keep], gx[keep])


# ---------------------------------------------------------------------------------------- straight from memory

# rows a wave (in sixteens) and waves that share K, of the products gate and up, y, dg and du, gx
STRAIGHT = [
    (F32, 16, 1024, 2736, 1024, "1/16"), (F32, 33, 129, 300, 129, "1/1"), (F32, 30, 1024, 2736, 1000, "2/8"), (F32, 64, 1000, 2736, 1024, "4/8"),
    (F32, 400, 512, 1376, 500, "2/1"), (F32, 3000, 130, 345, 120, "4/1"), (F32, 2000, 128, 344, 128, "2/1"), (F32, 130, 256, 680, 256, "1/8"),
    (BF16, 16, 1024, 2736, 1024, "1/16"), (BF16, 33, 129, 300, 129, "1/1"), (BF16, 30, 1024, 2736, 1000, "2/8"), (BF16, 80, 768, 1400, 768, "4/8"),
    (BF16, 40, 512, 1376, 512, "4/8"), (BF16, 3300, 32, 288, 31, "2/1"), (BF16, 6900, 32, 288, 32, "4/1"), (BF16, 130, 256, 680, 250, "1/8"),
]


def shapes(tmp_path, products):
    calls = "\n".join(f'  f = dp_form({n}, {m}, {k}, {parts}, {unit}); std::printf("%d/%d ", f.mt, f.wk);' for n, m, k, parts, unit in products)
    return run_host(tmp_path, f'#include <cstdio>\n#include "direct_shape.h"\nint main() {{\n  DpForm f;\n{calls}\n}}\n').split()


def test_the_sizes_take_every_straight_form(tmp_path):
    products, used = [], []
    for dtype, rows, width, hidden, out, form in STRAIGHT:
        way = forms(is_bf16(dtype), rows, width, hidden, out)
        assert way[0] == "straight", (rows, width, hidden, out)
        mine = [(hidden, rows, width, 1, 32), (out, rows, hidden, 1, 32)]
        if way[1] == "straight":
            mine += [(hidden, rows, out, 1, 32), (width, rows, hidden, 2, 32)]
        products += mine
        used += [(is_bf16(dtype), i, form) for i in range(len(mine))]
    found = set()
    for got, (bf16, i, form) in zip(shapes(tmp_path, products), used):
        found.add((bf16, i < 2, got))
    listed = {(is_bf16(dtype), form) for dtype, *_, form in STRAIGHT}
    assert listed <= {(bf16, got) for bf16, _, got in found}
    assert {got for _, _, got in found} == {"1/1", "1/8", "1/16", "2/1", "2/8", "4/1", "4/8"}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,hidden,out", [size[:5] for size in STRAIGHT])
def test_straight(dtype, rows, width, hidden, out):
    check(*make(rows, width, hidden, out, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,out", [(16, 4096, 1024), (32, 2048, 1024), (64, 2048, 1000), (1000, 500, 600), (2000, 300, 500), (500, 200, 100), (130, 1024, 100)])
def test_8_bit_products_straight(rows, width, out, dtype):
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows
    from test_int8 import make as rows_of

    x, w = rows_of(rows, width, dtype), rows_of(out, width, F32, seed=1)
    y = linear_int8(x.cuda(), quantize_rows(w.cuda()))
    oracle.near(y, *oracle.linear_int8(*oracle.quantize(x), *oracle.quantize(w), None, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,out", [(2000, 1024, 1024), (3000, 600, 2000), (5000, 515, 1030), (700, 3000, 1500), (9000, 300, 300)])
def test_8_bit_products_in_tiles(rows, width, out, dtype):
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows
    from test_int8 import make as rows_of

    assert rows * width * out > 4e8
    x, w = rows_of(rows, width, dtype), rows_of(out, width, F32, seed=1)
    y = linear_int8(x.cuda(), quantize_rows(w.cuda()))
    oracle.near(y, *oracle.linear_int8(*oracle.quantize(x), *oracle.quantize(w), None, dtype))


def test_8_bit_products_take_every_straight_form(tmp_path):
    from fastmd_amd import _abi

    sizes = [(16, 4096, 1024), (32, 2048, 1024), (64, 2048, 1000), (1000, 500, 600), (2000, 300, 500), (500, 200, 100), (130, 1024, 100)]
    for rows, width, out in sizes:
        assert _abi.load().fmd_linear_int8_work_size(1, rows, width, out) == 0
        assert rows * width * out <= 4e8 and width * out <= 2.5e7
    assert shapes(tmp_path, [(out, rows, -(-width // 16) * 16, 1, 64) for rows, width, out in sizes]) == [
        "1/16", "2/8", "4/8", "2/1", "4/1", "1/1", "1/8"]


def test_no_size_that_the_checks_accept_has_too_many_tiles():
    """Just below each limit of the argument checks (2^29 rows, 2^36 values of a matrix): sizes are found, which a refused call has none of."""
    from fastmd_amd import _abi
    from fastmd_amd.ops import feed_forward as ff

    lib = _abi.load()
    for hidden, width in ((129, 136), (257, 128), (128, 260), (1025, 100), (700, 2 ** 14 + 1), (2 ** 18 - 1, 2 ** 18 - 1)):
        widest = max(hidden, width)
        rows = min(ff.MAX_ROWS - 1, (ff.MAX_VALUES - 1) // widest)
        assert max(rows, widest) * widest < ff.MAX_VALUES
        for bf16 in (0, 1):
            assert forms(bf16, rows, width, hidden, width) == ("tiles", "tiles")
            assert lib.fmd_gated_ffn_work_size(bf16, rows, width, hidden, width, 15, 0) > 0
            assert lib.fmd_gated_ffn_bwd_work_size(bf16, rows, width, hidden, width, 15, 1, 1) > 0
