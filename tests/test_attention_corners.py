"""(g) Corners of segment attention and of the norm with rotation."""
import pytest
import torch

from test_attention import TYPES


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads,dim", [(40000, 4, 32), (2000, 8, 64), (9000, 4, 128)])
def test_many_queries_without_keys(rows, heads, dim, dtype):
    """Enough queries for every shape of tile, and no key row at all: zeros, and zero gradients."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    q = torch.ones(rows, heads, dim, dtype=dtype, device="cuda")
    k = torch.ones(0, heads, dim, dtype=dtype, device="cuda")
    q_off, k_off = torch.tensor([0, rows], device="cuda"), torch.tensor([0, 0], device="cuda")
    out, saved = segment_attention_forward(q, k, k, q_off, k_off)
    assert not out.any() and bool((saved.lse == -float("inf")).all())
    gq, gk, gv = segment_attention_vjp(q, q, k, k, out, saved, q_off, k_off)
    assert not gq.any() and gk.shape == gv.shape == (0, heads, dim)
