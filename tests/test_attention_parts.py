"""(g) Either half of the VJP of segment attention alone: the same bits as together, and None for the other."""
import pytest
import torch

from test_attention import TYPES, make


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,lk,heads,kv_heads,dim", [
    ([40, 0, 33], [50, 9, 0], 4, 2, 32),          # narrow tiles
    ([1900, 1900], [1900, 1900], 8, 8, 64),       # wide
    ([900, 700], [900, 650], 4, 4, 64),           # middle ones of float32
    ([3, 2], [6000, 4000], 16, 4, 128),           # split keys
    ([2000], [300], 8, 1, 64),                    # split queries
    ([1] * 300, [20] * 300, 4, 4, 32),            # the row kernels: one pass
    ([1] * 300, [20] * 300, 6, 2, 40),            # and a pass per head
    ([0, 90] + [1] * 200, [5, 200] + [7] * 200, 4, 2, 32),  # with a long segment
])
def test_halves_alone(lq, lk, heads, kv_heads, dim, dtype):
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    q, k, v, g, q_off, k_off = (x.cuda() for x in make(lq, lk, heads, kv_heads, dim, dtype, before=2, after=3))
    for causal in (False, True):
        out, saved = segment_attention_forward(q, k, v, q_off, k_off, causal=causal)
        half = lambda **need: segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off, causal=causal, **need)  # noqa: E731
        gq, gk, gv = half()
        only_q, no_k, no_v = half(need_kv=False)
        assert no_k is None and no_v is None and torch.equal(only_q, gq)
        no_q, only_k, only_v = half(need_q=False)
        assert no_q is None and torch.equal(only_k, gk) and torch.equal(only_v, gv)
        assert half(need_q=False, need_kv=False) == (None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_autograd_asks_for_what_is_wanted(wanted):
    from fastmd_amd.ops.attention import segment_attention

    q, k, v, g, off, _ = (x.cuda() for x in make([70, 33], [70, 33], 4, 2, 32, torch.float32))
    full = [x.clone().requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(segment_attention(*full, off), full, g)
    some = [x.clone().requires_grad_(n in wanted) for n, x in enumerate((q, k, v))]
    got = torch.autograd.grad(segment_attention(*some, off), [some[n] for n in wanted], g)
    for n, x in zip(wanted, got):
        assert torch.equal(x, want[n])
