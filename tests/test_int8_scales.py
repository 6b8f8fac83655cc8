"""(h) The 8-bit product's scales and bias: each result is the exact one rounded to float32 (and from there to bfloat16), whatever the
sizes of the two scales are apart. float64 leaves three roundings of 2^-53 of the scaled sum and the bias: 2^-50 of their
absolute values covers them."""
import pytest
import torch

from oracle import blocks as oracle

SIZES = [(3, 64, 40), (16, 4096, 64), (1000, 4096, 130)]  # the last in tiles


def check(q, scale, w, w_scale, bias, kind):
    from fastmd_amd.ops.int8 import Int8Rows, linear_int8

    y = linear_int8(Int8Rows(q.cuda(), scale.cuda()), Int8Rows(w.cuda(), w_scale.cuda()), None if bias is None else bias.cuda(), dtype=kind)
    s = (q.double() @ w.double().T) * scale.double()[:, None] * w_scale.double()
    want = s if bias is None else s + bias.double()
    terms = s.abs() + (0 if bias is None else bias.double().abs())
    smallest = 2.0 ** -150  # half of float32's smallest step
    bound = 2.0 ** -24 * want.abs() + (oracle.rounding(kind) * want.abs() * (1 + 2.0 ** -24) if kind == torch.bfloat16 else 0)
    got = y.double().cpu()
    assert bool(torch.isfinite(got).all())
    assert bool(((got - want).abs() <= bound + 2.0 ** -50 * terms + smallest).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width,out", SIZES)
@pytest.mark.parametrize("row,column", [(1e33, 1e-12), (1e-12, 1e33), (3e-44, 1e30), (1e30, 3e-44), (0.01, 0.02)])
def test_scales_of_different_sizes(row, column, rows, width, out, kind):
    g = torch.Generator().manual_seed(rows)
    q, w = (torch.randint(-127, 128, (n, width), generator=g, dtype=torch.int8) for n in (rows, out))
    q[:2], w[:2] = 127, 127  # the largest sums
    scale, w_scale = (f * (1 + torch.rand(n, generator=g)) for f, n in ((row, rows), (column, out)))
    check(q, scale, w, w_scale, None, kind)
    typical = float(row * column * 5e3 * width ** 0.5)
    check(q, scale, w, w_scale, torch.randn(out, generator=g) * typical, kind)


@pytest.mark.gpu
def test_a_bias_that_takes_the_sum_away():
    """What is left of sum and bias is exact to its own last bit."""
    q, w = torch.full((4, 64), 127, dtype=torch.int8), torch.full((8, 64), 127, dtype=torch.int8)
    scale, w_scale = torch.full((4,), 1 / 3), torch.full((8,), 1 / 7)
    total = (127 * 127 * 64 * scale.double()[0] * w_scale.double()[0]).float()
    check(q, scale, w, w_scale, -total.expand(8).contiguous(), torch.float32)
