"""(g) Norm and rotation of queries and keys: the HIP kernels against the definition in float64.

Error bounds (before any run). A float32 output is a sum of two products of a normalised value (relative error: the mean
square's, below 8 * 2^-24 over up to 256 squares in a tree, halved by the root, with division, root and two products: 10 * 2^-24)
and a table entry: 12 * 2^-24 of |a cos| + |b sin|, itself below the row's norm; a gradient adds the mean's dot product:
below 32 * 2^-24 of the same with absolute values. Row norms stand for the sums here. bf16 adds one rounding to 8 bits, 2^-8.
A weight's gradient adds over all rows: 2^-24 per term of their absolute sum, times 32 (a thread's run is at most 32 long
in these tests, trees above it), and the terms' own 32 * 2^-24.
"""
import math

import pytest
import torch

from oracle import attention as oracle

TYPES = [torch.float32, torch.bfloat16]


def tables(n, width, seed=0):
    from fastmd_amd.ops.qk_norm import rotary_tables

    return rotary_tables(n, width) if width else (torch.zeros(n, 0), torch.zeros(n, 0))


def near(got, want, scale, dtype, steps):
    got = got.double().cpu()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    tol = steps * 2.0 ** -24 * scale + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) * want.abs() + 1e-30
    worst = float(((got - want).abs() / tol).max()) if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.2f} of the bound"


def make(tokens, heads, kv_heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, f=1.0: (torch.randn(*s, generator=g) * f).to(dtype)  # noqa: E731
    return (r(tokens, heads, dim, f=2.0), r(tokens, kv_heads, dim, f=2.0), r(dim), r(dim), r(tokens, heads, dim),
            r(tokens, kv_heads, dim))


def check(q, k, wq, wk, gq, gk, cos, sin, positions, *, eps=1e-6, interleaved=False):
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, qk_norm_rotary_vjp

    cuda = lambda *xs: [None if x is None else x.cuda() for x in xs]  # noqa: E731
    args = cuda(q, k, wq, wk, cos, sin, positions)
    kw = {"eps": eps, "interleaved": interleaved}
    out = qk_norm_rotary(*args, **kw)
    grads = qk_norm_rotary_vjp(*cuda(gq, gk), *args, **kw)
    for n, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        y, gx, gw = oracle.norm_rotary(x, w, cos, sin, positions, eps=eps, interleaved=interleaved, g=g)
        d = x.shape[-1]
        near(out[n], y, y.norm(dim=-1, keepdim=True), x.dtype, 12)
        weight = torch.ones(d).double() if w is None else w.double()
        rms = torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)
        size = (g.double().norm(dim=-1, keepdim=True) * float(weight.abs().max()) / rms * 2)
        near(grads[n], gx, size, x.dtype, 32)
        if w is None:
            assert grads[2 + n] is None
            continue
        terms = (g.double().norm(dim=-1, keepdim=True) * (x.double() / rms).norm(dim=-1, keepdim=True)).sum()
        near(grads[2 + n], gw, terms.expand(d), x.dtype, 64)
    return out, grads


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot", [(8, 8), (8, 2), (16, 16), (32, 32), (40, 40), (40, 26), (64, 0), (64, 32), (96, 96),
                                     (128, 64), (128, 128), (128, 48), (200, 200), (256, 256)])
def test_widths(dim, rot, dtype, interleaved):
    q, k, wq, wk, gq, gk = make(37, 5, 2, dim, dtype, seed=dim + rot)
    cos, sin = tables(50, rot)
    positions = torch.randint(0, 50, (37,), generator=torch.Generator().manual_seed(1))
    check(q, k, wq, wk, gq, gk, cos, sin, positions, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 16, 4), (3, 7, 1), (135, 4, 4), (2500, 9, 3)])
def test_sizes(tokens, heads, kv_heads, dtype):
    q, k, wq, wk, gq, gk = make(tokens, heads, kv_heads, 64, dtype, seed=tokens)
    cos, sin = tables(tokens, 64)
    check(q, k, wq, wk, gq, gk, cos, sin, None)
    check(q, k, None, wk, gq, gk, cos, sin, torch.arange(tokens, dtype=torch.int32).flip(0), eps=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_zero_rows(dtype):
    """A row of zeros has the norm of eps: output zero, gradient g w / sqrt(eps)."""
    q, k, wq, wk, gq, gk = make(6, 2, 2, 32, dtype)
    q[2] = 0.0
    cos, sin = tables(6, 32)
    out, grads = check(q, k, wq, wk, gq, gk, cos, sin, None, eps=1e-4)
    assert not out[0][2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(dtype):
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, qk_norm_rotary_vjp

    q, k, wq, wk, gq, gk = (x.cuda() for x in make(33, 4, 2, 32, dtype))
    cos, sin = (x.cuda() for x in tables(33, 32))
    want = (*qk_norm_rotary(q, k, wq, wk, cos, sin), *qk_norm_rotary_vjp(gq, gk, q, k, wq, wk, cos, sin))
    packed, gpacked = torch.cat((q, k, k), 1), torch.cat((gk, gq), 1)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    wide = torch.zeros(40, 20, device="cuda")
    c2, s2 = wide.clone()[:33, 3:19].copy_(cos), wide.clone()[:33, 3:19].copy_(sin)
    w_odd = torch.empty(33, dtype=dtype, device="cuda")[1:].copy_(wq)
    for args, grads in (((packed[:, :4], packed[:, 4:6], wq, wk, cos, sin), (gpacked[:, 2:], gpacked[:, :2])),
                        ((odd, k, w_odd, wk, c2, s2), (gq, gk))):
        got = (*qk_norm_rotary(*args), *qk_norm_rotary_vjp(*grads, *args))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_alone(dtype, interleaved):
    """The turn keeps each pair's length; turning back by the other sign gives the input; the gradient is that."""
    from fastmd_amd.ops.qk_norm import rotary, rotary_tables

    x = make(50, 3, 1, 64, dtype)[0].cuda()
    cos, sin = rotary_tables(200, 48, device="cuda")
    positions = torch.randint(0, 200, (50,), device="cuda")
    y = rotary(x, cos, sin, positions, interleaved=interleaved)
    want = oracle.norm_rotary(x.cpu(), None, cos.cpu(), sin.cpu(), positions.cpu(), interleaved=interleaved,
                              norm=False)[0]
    near(y, want, want.norm(dim=-1, keepdim=True), dtype, 4)
    assert torch.equal(y[..., 48:], x[..., 48:])
    back = rotary(y, cos, -sin, positions, interleaved=interleaved)
    near(back, x.double().cpu(), x.double().cpu().norm(dim=-1, keepdim=True), torch.float32,
         8 if dtype == torch.float32 else 2 ** 17)
    a = x.clone().requires_grad_()
    g = torch.randn(x.shape, device="cuda").to(dtype)
    rotary(a, cos, sin, positions, interleaved=interleaved).backward(g)
    assert torch.equal(a.grad, rotary(g, cos, -sin, positions, interleaved=interleaved))


@pytest.mark.gpu
def test_autograd_against_differences():
    from fastmd_amd.ops.qk_norm import qk_norm_rotary

    q, k, wq, wk, gq, gk = make(9, 3, 2, 24, torch.float32, seed=4)
    cos, sin = tables(9, 16)
    leaves = [x.cuda().requires_grad_() for x in (q, k, wq, wk)]
    a, b = qk_norm_rotary(*leaves, cos.cuda(), sin.cuda())
    ((a * gq.cuda()).sum() + (b * gk.cuda()).sum()).backward()
    gen = torch.Generator().manual_seed(2)
    for n in range(4):
        way = torch.randn(leaves[n].shape, generator=gen).double()
        value = []
        for step in (1e-5, -1e-5):
            x = [t.double() for t in (q, k, wq, wk)]
            x[n] = x[n] + step * way
            value.append(sum(float((oracle.norm_rotary(x[i], x[2 + i], cos, sin)[0] * g.double()).sum())
                             for i, g in enumerate((gq, gk))))
        want, got = (value[0] - value[1]) / 2e-5, float((leaves[n].grad.double().cpu() * way).sum())
        assert abs(got - want) <= 1e-5 * float((leaves[n].grad.double().cpu() * way).abs().sum())


@pytest.mark.gpu
def test_one_output_used():
    """The other output's gradient is none: zero."""
    from fastmd_amd.ops.qk_norm import qk_norm_rotary

    q, k, wq, wk, gq, gk = (x.cuda() for x in make(9, 3, 2, 24, torch.float32))
    cos, sin = (x.cuda() for x in tables(9, 16))
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    qk_norm_rotary(*leaves, cos, sin)[0].backward(gq)
    assert leaves[0].grad.any() and leaves[2].grad.any() and not leaves[1].grad.any() and not leaves[3].grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_outside_the_table(dtype):
    from fastmd_amd.ops.qk_norm import rotary

    x = torch.ones(4, 2, 16, device="cuda")
    cos, sin = (t.cuda() for t in tables(3, 8))
    y = rotary(x, cos, sin, torch.tensor([0, 3, -1, 2], dtype=dtype, device="cuda"))
    assert torch.isnan(y[1:3, :, :8]).all() and torch.isfinite(y[1:3, :, 8:]).all()
    assert torch.isfinite(y[[0, 3]]).all()


@pytest.mark.gpu
def test_repeatable_weight_gradients():
    from fastmd_amd.ops.qk_norm import qk_norm_rotary_vjp

    q, k, wq, wk, gq, gk = (x.cuda() for x in make(3000, 8, 8, 64, torch.float32))
    cos, sin = (x.cuda() for x in tables(3000, 64))
    runs = [qk_norm_rotary_vjp(gq, gk, q, k, wq, wk, cos, sin) for _ in range(2)]
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_no_tokens():
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, qk_norm_rotary_vjp

    q, k, w = torch.ones(0, 4, 32, device="cuda"), torch.ones(0, 2, 32, device="cuda"), torch.ones(32, device="cuda")
    cos, sin = (x.cuda() for x in tables(3, 32))
    a, b = qk_norm_rotary(q, k, w, w, cos, sin)
    assert a.shape == q.shape and b.shape == k.shape
    grads = qk_norm_rotary_vjp(q, k, q, k, w, w, cos, sin)
    assert not grads[2].any() and not grads[3].any()


@pytest.mark.gpu
def test_rows_past_32_bits():
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, qk_norm_rotary_vjp

    tokens = 2 ** 31 // 2048 + 70
    q, k, _, _, gq, gk = make(70, 16, 1, 128, torch.bfloat16)
    cos, sin = tables(100, 128)

    def last(x):
        y = torch.empty(tokens, *x.shape[1:], dtype=x.dtype, device="cuda")
        y[-70:] = x.cuda()
        return y

    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") % 100
    args = (last(q), last(k), None, None, cos.cuda(), sin.cuda(), positions)
    out = qk_norm_rotary(*args)
    grads = qk_norm_rotary_vjp(last(gq), last(gk), *args)
    at = positions[-70:].cpu()
    for n, (x, g) in enumerate(((q, gq), (k, gk))):
        y, gx, _ = oracle.norm_rotary(x, None, cos, sin, at, g=g)
        near(out[n][-70:], y, y.norm(dim=-1, keepdim=True), x.dtype, 12)
        rms = torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6)
        near(grads[n][-70:], gx, g.double().norm(dim=-1, keepdim=True) / rms * 2, x.dtype, 32)


@pytest.mark.gpu
def test_refusals():
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, qk_norm_rotary_vjp, rotary

    q, k, w = torch.ones(5, 4, 32, device="cuda"), torch.ones(5, 2, 32, device="cuda"), torch.ones(32, device="cuda")
    cos, sin = (x.cuda() for x in tables(5, 32))
    at = torch.arange(5, device="cuda")
    bad = [
        (lambda: qk_norm_rotary(q[0], k, w, w, cos, sin), "tokens, heads, dim"),
        (lambda: qk_norm_rotary(q.half(), k.half(), w, w, cos, sin), "float32 or bfloat16"),
        (lambda: qk_norm_rotary(q, k.bfloat16(), w, w, cos, sin), "float32 or bfloat16"),
        (lambda: qk_norm_rotary(q, k[:4], w, w, cos, sin), "share tokens"),
        (lambda: qk_norm_rotary(q, k, w[:16], w, cos, sin), "q_weight"),
        (lambda: qk_norm_rotary(q, k, w, w.bfloat16(), cos, sin), "k_weight"),
        (lambda: qk_norm_rotary(q, k, w, w, cos, sin[:, :8]), "one shape"),
        (lambda: qk_norm_rotary(q, k, w, w, cos.double(), sin.double()), "float32 tables"),
        (lambda: qk_norm_rotary(q[..., :16], k[..., :16], None, None, cos, sin), "columns"),
        (lambda: qk_norm_rotary(q, k, w, w, cos[:4], sin[:4]), "rows for 5 tokens"),
        (lambda: qk_norm_rotary(q, k, w, w, cos, sin, at[:4]), "positions"),
        (lambda: qk_norm_rotary(q, k, w, w, cos, sin, at.float()), "positions"),
        (lambda: qk_norm_rotary(q, k, w, w, cos, sin, eps=-1.0), "eps"),
        (lambda: qk_norm_rotary(q[..., :12], k[..., :12], None, None, cos[:, :4], sin[:, :4]), "multiple of 8"),
        (lambda: qk_norm_rotary_vjp(q[:, :3], k, q, k, w, w, cos, sin), "gq"),
        (lambda: rotary(q.cpu(), cos, sin), "GPU"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_tables():
    """Angles of the definition; a stretched context keeps the fast pairs and slows the slow ones by its factor."""
    from fastmd_amd.ops.qk_norm import rotary_frequencies, rotary_tables

    cos, sin = rotary_tables(5, 8)
    assert cos.shape == (5, 4) and cos.dtype == torch.float32
    assert float(cos[3, 1]) == pytest.approx(math.cos(3 * 10000.0 ** -0.25), abs=1e-7)
    assert float(sin[4, 0]) == pytest.approx(math.sin(4.0), abs=1e-7)
    f = rotary_frequencies(64)
    assert torch.allclose(rotary_frequencies(64, factor=4.0), f / 4)
    g = rotary_frequencies(64, factor=8.0, trained_length=2048)
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 4], f[turns >= 4]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and bool(((g < f) & (g > f / 8))[mid].all())
    c2, _ = rotary_tables(torch.tensor([0.5, 7.25]), 8, amplitude=1.5)
    assert float(c2[1, 0]) == pytest.approx(1.5 * math.cos(7.25), abs=1e-6)
    for bad in (dict(width=7), dict(width=0), dict(width=8, base=-1.0), dict(width=8, factor=0.0),
                dict(width=8, factor=2.0, trained_length=16, low=4.0, high=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_cpu_tensors_are_refused():
    from fastmd_amd.ops.qk_norm import rotary

    with pytest.raises(ValueError, match="GPU"):
        rotary(torch.zeros(2, 1, 8), torch.zeros(2, 4), torch.zeros(2, 4))


def test_entry_points_refuse_what_no_launch_can_honour():
    from fastmd_amd import _abi

    lib = _abi.load()
    call = lambda **kw: lib.fmd_qk_norm_rotary(  # noqa: E731
        0, 16, 32, 32, 1, None, 0, 0, 0, kw.get("tokens", 4), kw.get("dim", 32), 1, 1e-6, None, None, 16, 16,
        kw.get("rows", 4), 16, kw.get("rot", 32), 0, None, 0, 16, None, None)
    assert call(rot=31) == 10001 and call(rot=64) == 10001 and call(rows=3) == 10001 and call(tokens=-1) == 10001
    assert call(dim=36) == 10002 and call(dim=264) == 10002
