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
