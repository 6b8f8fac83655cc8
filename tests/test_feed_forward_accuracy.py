"""(h) The gated feed-forward block in bfloat16: every result is as near to the exact one as rounding it once allows.

A result x (1 + e) rounded to bf16 is off by the rounding's error and by e, which add up as independent errors do:
sqrt(1 + (e / r)^2) times the rounding's alone, whose root mean square is r = 2^-7 / sqrt(12) of the power of two below x, 1.6e-3 of x over
a spread of sizes. What the kernels leave of e: h, dg and du in 16 bits (two parts of 8: at most 2^-17 of each), float32 sums of n terms
(sqrt(n) 2^-24 in the root mean square of terms of either sign: 2^-18 for 4 096), the activation (some 2^-24). Together below 2e-5: a
ratio of 1.0001. The bound is 1.01. Operands of one part bring e to r, and the ratio to 1.4."""
import pytest
import torch

from feed_forward_forms import forms
from oracle import blocks as oracle
from test_feed_forward import make

BOUND = 1.01
SIZES = [  # forms of the forward pass and of the VJP
    (33, 40, 100, 40, "one", "one"),            # units of K past the hidden width
    (135, 64, 128, 64, "one", "one"),
    (8200, 64, 120, 64, "one", "one"),          # 32 rows of a workgroup
    (1, 512, 1376, 512, "straight", "straight"),
    (16, 512, 1376, 512, "straight", "straight"),
    (40, 333, 517, 209, "straight", "straight"),
    (130, 256, 680, 256, "straight", "straight"),
    (16, 1024, 2736, 1024, "straight", "tiles"),
    (1500, 301, 1003, 299, "tiles", "tiles"),   # odd widths: every operand laid out
    (2100, 512, 1376, 512, "tiles", "tiles"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,hidden,out,forward,back", SIZES)
def test_results_are_rounded_once(rows, width, hidden, out, forward, back):
    from fastmd_amd.ops.feed_forward import gated_feed_forward, gated_feed_forward_forward, gated_feed_forward_vjp

    x, wg, wu, wd, gy = make(rows, width, hidden, out, torch.bfloat16, seed=11)
    want = [value for value, _ in oracle.gated(x, wg, wu, wd, "silu", gy)]
    x, wg, wu, wd, gy = (t.cuda() for t in (x, wg, wu, wd, gy))
    y, saved = gated_feed_forward_forward(x, wg, wu, wd)
    got = (y, *gated_feed_forward_vjp(gy, x, wg, wu, wd, saved))
    assert torch.equal(gated_feed_forward(x, wg, wu, wd), y)
    for name, t, w in zip(("y", "gx", "g_gate", "g_up", "g_down"), got, want):
        once = float((w.bfloat16().double() - w).square().sum().sqrt())
        ratio = float((t.double().cpu() - w).square().sum().sqrt()) / once
        assert ratio <= BOUND, f"{name}: {ratio:.3f} times the error of rounding the exact result"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,hidden,out", [size[:4] for size in SIZES if size[0] in (33, 40, 2100)])
def test_an_infinite_hidden_value_stays_infinite(rows, width, hidden, out):
    """Its second part is zero, not the difference of infinities."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward

    x, wg, wu, wd, _ = (t.cuda() for t in make(rows, width, hidden, out, torch.bfloat16))
    wg[:, 0], wu[:, 0], x[:, 0] = 0.0, 0.0, 0.0
    wg[5, 0], wu[5, 0] = 1.0, 1.0
    want = gated_feed_forward(x, wg, wu, wd)
    x[3] = 0.0
    x[3, 0] = 2.0 ** 100
    y = gated_feed_forward(x, wg, wu, wd)
    assert torch.equal(y[3], torch.sign(wd[:, 5]) * float("inf"))
    assert torch.equal(y[:3], want[:3]) and torch.equal(y[4:], want[4:])


def test_the_sizes_take_every_form():
    for rows, width, hidden, out, forward, back in SIZES:
        assert forms(1, rows, width, hidden, out) == (forward, back), (rows, width, hidden, out)
