"""(h) The gated feed-forward block in float32, whose operands go through the matrix cores in three planes of 8 bits: results that are
exact only if every plane product is there, and the size of the rounding errors.

Exact: operands of whole numbers, one of them of 22 bits (all three planes), the others 0 and +-1, or two of 11 bits (the product of the
two second planes). Where the absolute values of a result's terms sum up to less than 2^23, every plane product and every sum of
them in any order is a whole number below 2^24, and the result has to be equal. Other results are left out.

Errors: a float32 sum of n terms of either sign in six plane products is rounded at most 6 n times, each time by 0.41 2^-24 of what has
been summed in the root mean square, which grows as the root of the number of terms up to T, the root of the terms' squares:
0.29 sqrt(6 n) 2^-24 T, and at most 2^-24 T for products that are left out and the last rounding. h and the gradients of the
projections carry the like of two such sums each (2.5 times one covers the activation's slope of at most 1.1, and its
own error). A bound of 1.5 times that is 10^3 times below the error of products of one plane, 10 times below that of two."""
import math

import pytest
import torch

from feed_forward_forms import forms
from oracle import blocks as oracle
from test_feed_forward import make

SIZES = [(135, 64, 128, 64, "one"), (130, 256, 680, 256, "straight"), (400, 512, 1376, 500, "straight"), (2100, 304, 520, 312, "tiles"),
         (1500, 301, 1003, 299, "tiles")]


def whole(case, rows, width, hidden, out):
    g = torch.Generator().manual_seed(len(case) + rows)
    sign = lambda *s: 1 - 2 * torch.randint(0, 2, s, generator=g)  # noqa: E731
    many = lambda bits, *s: torch.randint(2 ** (bits - 1), 2 ** bits, s, generator=g) * sign(*s)  # noqa: E731

    def one_each(r, c, values, first=0):
        """A value in each row, at any column from `first` on."""
        m = torch.zeros(r, c, dtype=torch.int64)
        m[torch.arange(r), torch.randint(first, c, (r,), generator=g)] = values
        return m

    x, wg, wu = torch.zeros(rows, width, dtype=torch.int64), torch.zeros(hidden, width, dtype=torch.int64), torch.zeros(hidden, width, dtype=torch.int64)
    x[:, 0], wu[:, 0] = 1, sign(hidden)  # the second projection is 1 or -1
    wd, gy = one_each(out, hidden, sign(out)), torch.zeros(rows, out, dtype=torch.int64)
    n = min(rows, out)
    gy[:n] = torch.diag(sign(n))[:, torch.randperm(n, generator=g)] if n == out else torch.eye(n, out, dtype=torch.int64) * sign(n, 1)
    if case == "rows":
        x[:, 1:], wg = many(22, rows, width - 1), one_each(hidden, width, sign(hidden), 1)
    elif case == "gate":
        x[:, 1:], wg[:, 1:] = one_each(rows, width, sign(rows), 1)[:, 1:], many(22, hidden, width - 1)
    elif case == "down":
        x[:, 1:], wg[:, 0] = one_each(rows, width, sign(rows), 1)[:, 1:], sign(hidden)
        wd = one_each(out, hidden, many(22, out))
    elif case == "gradient":
        x[:, 1:], wg[:, 0] = one_each(rows, width, sign(rows), 1)[:, 1:], sign(hidden)
        wg[:, 1:] = one_each(hidden, width, sign(hidden), 1)[:, 1:]
        gy = gy * many(22, rows, 1)
        x[n:, 1:] = 0
    elif case == "both":
        x[:, 1:], wg[:, 1:] = one_each(rows, width, many(11, rows), 1)[:, 1:], many(11, hidden, width - 1)
    elif case == "both last":
        x[:, 1:], wg[:, 1:] = one_each(rows, width, many(11, rows), 1)[:, 1:], sign(hidden, width - 1)
        wd = one_each(out, hidden, many(11, out))
    return [t.double() for t in (x, wg, wu, wd, gy)]


def product(a, b, bad_a=None, bad_b=None):
    """a b, and where it is exact: terms below 2^23 in all, none of them of a factor that is not exact itself."""
    terms, some = a.abs() @ b.abs(), lambda t: (t != 0).double()  # noqa: E731
    bad = terms >= 2.0 ** 23
    if bad_a is not None:
        bad |= (bad_a.double() @ some(b)) > 0
    if bad_b is not None:
        bad |= (some(a) @ bad_b.double()) > 0
    return a @ b, bad


# results that reach the planes of each case's large operand
TELLING = {"rows": ("y", "g_up", "g_down"), "gate": ("y", "gx", "g_up", "g_down"), "down": ("y", "gx", "g_gate", "g_up"),
           "gradient": ("gx", "g_gate", "g_down"), "both": ("y", "g_up", "g_down"), "both last": ("y", "g_up")}


def expected(x, wg, wu, wd, gy):
    """{name: (value, where it is exact)} without an activation"""
    g, bad_g = product(x, wg.T)
    u, bad_u = product(x, wu.T)
    h, gh = g * u, None
    bad_h = bad_g | bad_u | (h.abs() >= 2.0 ** 23)
    gh, bad_gh = product(gy, wd)
    dg, du = gh * u, gh * g
    bad_dg, bad_du = bad_gh | ((bad_u | (dg.abs() >= 2.0 ** 23)) & (gh != 0)), bad_gh | ((bad_g | (du.abs() >= 2.0 ** 23)) & (gh != 0))
    out = {"y": product(h, wd.T, bad_h)}
    a, bad_a = product(dg, wg, bad_dg)
    b, bad_b = product(du, wu, bad_du)
    out["gx"] = (a + b, bad_a | bad_b | (dg.abs() @ wg.abs() + du.abs() @ wu.abs() >= 2.0 ** 23))
    out["g_gate"] = product(dg.T, x, bad_dg.T)
    out["g_up"] = product(du.T, x, bad_du.T)
    out["g_down"] = product(gy.T, h, None, bad_h)
    return {name: (value, ~bad) for name, (value, bad) in out.items()}


def test_enough_results_are_exact():
    for rows, width, hidden, out, form in SIZES:
        assert forms(0, rows, width, hidden, out)[0] == form
        for case, names in TELLING.items():
            want = expected(*whole(case, rows, width, hidden, out))
            for name in names:
                value, exact = want[name]
                large = (value[exact].abs() >= 2.0 ** (9 if name == "g_gate" and case == "down" else 17)).sum()
                assert int(large) >= 20, (case, name, rows, int(large))


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(TELLING))
@pytest.mark.parametrize("rows,width,hidden,out,form", SIZES)
def test_every_plane_product_is_there(rows, width, hidden, out, form, case):
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    args = whole(case, rows, width, hidden, out)
    x, wg, wu, wd, gy = (t.float().cuda() for t in args)
    y, saved = gated_feed_forward_forward(x, wg, wu, wd, activation=None)
    grads = gated_feed_forward_vjp(gy, x, wg, wu, wd, saved, activation=None)
    for (name, (value, exact)), got in zip(expected(*args).items(), (y, *grads)):
        assert torch.equal(got.double().cpu()[exact], value[exact]), name


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,hidden,out,form", SIZES)
def test_rounding_errors(rows, width, hidden, out, form):
    from fastmd_amd.ops.feed_forward import gated_feed_forward_forward, gated_feed_forward_vjp

    args = make(rows, width, hidden, out, torch.float32, seed=5)
    x, wg, wu, wd, gy = (t.double() for t in args)
    want = [value for value, _ in oracle.gated(*args[:4], "silu", args[4])]
    g, u = x @ wg.T, x @ wu.T
    a, d = oracle.act(g, "silu")
    gh = gy @ wd
    h, dg, du = a * u, gh * u * d, gh * a
    squares = [(h ** 2) @ (wd ** 2).T, (dg ** 2) @ wg ** 2 + (du ** 2) @ wu ** 2, (dg ** 2).T @ x ** 2, (du ** 2).T @ x ** 2, (gy ** 2).T @ h ** 2]
    sum_of = lambda n: 0.29 * math.sqrt(6 * n) + 1  # noqa: E731
    first, last = sum_of(max(width, out)), (hidden, 2 * hidden, rows, rows, rows)
    x, wg, wu, wd, gy = (t.cuda() for t in args)
    y, saved = gated_feed_forward_forward(x, wg, wu, wd)
    got = (y, *gated_feed_forward_vjp(gy, x, wg, wu, wd, saved))
    for name, t, w, s, n in zip(("y", "gx", "g_gate", "g_up", "g_down"), got, want, squares, last):
        error = float((t.double().cpu() - w).square().mean().sqrt() / s.mean().sqrt())
        bound = 1.5 * (2.5 * first + sum_of(n)) * 2.0 ** -24
        print(f"{form} {name}: {error * 2 ** 24:.2f} of {bound * 2 ** 24:.0f} units")
        assert error <= bound, f"{name}: {error * 2 ** 24:.1f} units, bound {bound * 2 ** 24:.1f}"
