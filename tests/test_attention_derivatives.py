"""Derivatives that the attention operators do not have raise, instead of missing from a result."""
import pytest
import torch

from fastmd_amd import systems
from fastmd_amd._autograd import first_derivatives


def test_gradients_that_kernels_form_cannot_be_differentiated_silently():
    """A function of the same form on the CPU: x^3 whose gradient is formed outside autograd."""

    class Cube(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.save_for_backward(x)
            return x.detach() ** 3

        @staticmethod
        def backward(ctx, g):
            (x,) = ctx.saved_tensors
            return first_derivatives("cube", (3.0 * g.detach() * x.detach() ** 2,), g, x)[0]

    x = torch.tensor(2.0, requires_grad=True)
    (first,) = torch.autograd.grad(Cube.apply(x), x)
    assert float(first) == 12.0 and not first.requires_grad
    (first,) = torch.autograd.grad(Cube.apply(x) + x ** 2, x, create_graph=True)
    assert float(first) == 16.0
    with pytest.raises(NotImplementedError, match="cube has first derivatives only"):
        first.backward()


def _leaves(*shapes):
    gen = torch.Generator().manual_seed(4)
    return [torch.randn(*s, generator=gen).cuda().requires_grad_() for s in shapes]


def _attention():
    from fastmd_amd.ops.attention import segment_attention

    leaves = _leaves((30, 4, 16), (30, 2, 16), (30, 2, 16))
    off = torch.tensor([0, 11, 30], device="cuda")
    return leaves, lambda q, k, v: segment_attention(q, k, v, off)


def _norm():
    from fastmd_amd.ops.qk_norm import qk_norm_rotary, rotary_tables

    tables = rotary_tables(9, 16, device="cuda")
    return (_leaves((9, 4, 16), (9, 2, 16), (16,), (16,)),
            lambda q, k, wq, wk: torch.cat(qk_norm_rotary(q, k, wq, wk, *tables), 1))


def _rotary():
    from fastmd_amd.ops.qk_norm import rotary, rotary_tables

    tables = rotary_tables(9, 16, device="cuda")
    return _leaves((9, 4, 16)), lambda x: rotary(x, *tables)


@pytest.mark.gpu
@pytest.mark.parametrize("weighted", [False, True])  # the gradient that comes in does not, or does, depend on the inputs
@pytest.mark.parametrize("operator", [_attention, _norm, _rotary])
def test_second_derivatives_raise(operator, weighted):
    leaves, call = operator()
    value = lambda: (call(*leaves) * (call(*leaves) if weighted else 1.0)).sum()  # noqa: E731
    plain = torch.autograd.grad(value(), leaves)
    grads = torch.autograd.grad(value(), leaves, create_graph=True)
    for a, b in zip(plain, grads):
        assert torch.equal(a, b)
    for g in grads:
        with pytest.raises(NotImplementedError, match="first derivatives only"):
            torch.autograd.grad((g ** 2).sum() + sum(x.sum() for x in leaves), leaves, retain_graph=True)


@pytest.mark.gpu
def test_a_loss_on_the_models_forces_raises(device):
    from fastmd_amd.models.attention_like import AttentionAdapter
    from test_attention_model import _builder

    s = systems.perovskite(2, sigma=0.2)
    adapter = AttentionAdapter(device=device)
    adapter.module.requires_grad_(True)
    builder = _builder(s, device)
    builder.build(torch.tensor(s.positions, device=device))
    positions = builder.batch.positions.detach().clone().requires_grad_()
    energy = adapter.node_energy(adapter.prepare(builder.batch), positions, builder.batch.cell).sum()
    (gradient,) = torch.autograd.grad(energy, positions, create_graph=True)
    with pytest.raises(NotImplementedError, match="first derivatives only"):
        (energy + (gradient ** 2).sum()).backward()


@pytest.mark.gpu
def test_second_derivatives_of_the_linear_layer(device):
    """A penalty on the input's gradient beside the value, against float64: sums of 40 products of order one, to 1e-5."""
    from fastmd_amd.ops.wide_gemm import linear

    def grads(x, w, b, layer):
        y = layer(x, w, b)
        value = (y ** 3).sum()
        (gx,) = torch.autograd.grad(value, x, create_graph=True)
        return gx, *torch.autograd.grad(0.1 * value + (gx ** 2).sum(), (x, w, b))

    gen = torch.Generator().manual_seed(6)
    data = [0.2 * torch.randn(*s, generator=gen) for s in ((50, 24), (40, 24), (40,))]
    want = grads(*[t.double().requires_grad_() for t in data], torch.nn.functional.linear)
    got = grads(*[t.to(device).requires_grad_() for t in data], linear)
    for a, b in zip(got, want):
        assert float((a.double().cpu() - b).abs().max()) < 1e-5 * float(b.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("operator", [_attention, _norm, _rotary])
def test_forward_mode_raises(operator):
    """An input with a tangent, none that wants a gradient; outside the dual level the call is as ever."""
    from torch.autograd import forward_ad

    leaves, call = operator()
    leaves = [x.detach() for x in leaves]
    want = call(*leaves)
    for n in range(len(leaves)):
        with forward_ad.dual_level():
            assert torch.equal(call(*leaves), want)
            dual = [forward_ad.make_dual(x, torch.ones_like(x)) if i == n else x for i, x in enumerate(leaves)]
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                call(*dual)
    assert torch.equal(call(*leaves), want)
