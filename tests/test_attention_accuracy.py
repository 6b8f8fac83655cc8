"""(g) Attention within segments in bfloat16: every result is as near to the exact one as rounding it once allows.

A result x (1 + e) rounded to bf16 is off by the rounding's error and by e, which add up as independent errors do:
sqrt(1 + (e / r)^2) times the rounding's alone, whose root mean square is r = 2^-7 / sqrt(12)
of the power of two below x, 1.6e-3 of x over a spread of sizes. What the kernels leave of e: weights of 16 bits (two parts of 8: at most 2^-17 of each), the part of
the output that delta takes in 16 bits (2^-17), scores with 2 * (16 * 2^-24 * S) for a largest absolute sum S (below 100 here: 2e-4 of a
weight at the most, 2e-5 in the root mean square, of which the few large sums make most). Together below 1e-4 in the root mean square: a ratio of
1.002 at the most. The bound is 1.01. Weights of one part would bring e to r, and the ratio to 1.4."""
import pytest
import torch

from oracle import attention as oracle
from test_attention import make

BOUND = 1.01


def ratios(lq, lk, heads, kv_heads, dim, causal, seed):
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    q, k, v, g, q_off, k_off = make(lq, lk, heads, kv_heads, dim, torch.bfloat16, seed=seed)
    r = oracle.segment_attention(q, k, v, q_off, k_off, causal=causal, gout=g)
    q, k, v, g, q_off, k_off = (x.cuda() for x in (q, k, v, g, q_off, k_off))
    out, saved = segment_attention_forward(q, k, v, q_off, k_off, causal=causal)
    got = (out, *segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off, causal=causal))
    result = {}
    for name, x in zip(("out", "gq", "gk", "gv"), got):
        want = r[name]
        once = float((want.bfloat16().double() - want).square().sum().sqrt())
        result[name] = float((x.double().cpu() - want).square().sum().sqrt()) / once
    return result


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk,heads,kv_heads,dim", [
    ([64] * 60, [64] * 60, 8, 8, 64),        # many small systems: the wide tiles, few keys each
    ([64], [64], 8, 8, 64),                  # one of them alone: the narrow ones
    ([1900, 1900], [1900, 1900], 8, 8, 32),  # wide, many keys; causal: few for the first rows
    ([1500, 300], [1500, 300], 16, 4, 128),  # wide, shared key heads
    ([900], [900], 16, 16, 96),
    ([245], [245], 24, 24, 16),              # narrow
    ([40, 7], [3000, 2100], 8, 2, 128),      # narrow rows over longer keys, split
    ([1] * 70, [9] * 70, 8, 2, 64),          # a query for each segment: the row kernels
])
def test_results_are_rounded_once(lq, lk, heads, kv_heads, dim, causal):
    for name, ratio in ratios(lq, lk, heads, kv_heads, dim, causal, seed=dim).items():
        assert ratio <= BOUND, f"{name}: {ratio:.3f} times the error of rounding the exact result"


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 64), (16, 4, 128)])
def test_first_rows_of_long_causal_sequences(heads, kv_heads, dim):
    """The rows that see few keys, in the tiles of calls with many."""
    from fastmd_amd.ops.attention import segment_attention_forward

    q, k, v, _, off, _ = make([1900, 1900], [1900, 1900], heads, kv_heads, dim, torch.bfloat16, seed=dim)
    out, _ = segment_attention_forward(*(x.cuda() for x in (q, k, v, off)), causal=True)
    for start in (0, 1900):
        few = slice(start, start + 60)  # causal: they see each other only
        want = oracle.segment_attention(q[few], k[few], v[few], [0, 60], [0, 60], causal=True)["out"]
        once = float((want.bfloat16().double() - want).square().sum().sqrt())
        assert float((out[few].double().cpu() - want).square().sum().sqrt()) <= BOUND * once


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk", [([64] * 60, [64] * 60), ([245], [245]), ([1] * 70, [9] * 70)])
def test_the_saved_residual_is_what_the_outputs_rounding_dropped(lq, lk):
    """out + residual has 16 bits of the exact output: 2^-16 of its size, and the weights' and scores' 2^-16 of the terms."""
    from fastmd_amd.ops.attention import segment_attention_forward

    q, k, v, _, q_off, k_off = make(lq, lk, 8, 8, 64, torch.bfloat16)
    r = oracle.segment_attention(q, k, v, q_off, k_off)
    out, saved = segment_attention_forward(*(x.cuda() for x in (q, k, v, q_off, k_off)))
    far = (out.double() + saved.residual.double()).cpu() - r["out"]
    assert bool((far.abs() <= 2.0 ** -16 * r["out"].abs() + 2.0 ** -15 * r["abs_out"] + 1e-30).all())
