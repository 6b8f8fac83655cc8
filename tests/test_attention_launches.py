"""(g) Attention and norm of more workgroups than one launch takes (2^32 threads), and what is too large for both."""
import pytest
import torch

from oracle import attention as oracle
from test_attention import U, bounds, compare, make


def _tail(lengths_q, lengths_k, segments, heads, dim, dtype):
    """Offsets of `segments` segments, all empty but the last few."""
    q, k, v, g, q_off, k_off = make(lengths_q, lengths_k, heads, heads, dim, dtype)
    empty = torch.zeros(segments - len(lengths_q), dtype=torch.int64)
    return (q, k, v, g, q_off, k_off), torch.cat((empty, q_off)).cuda(), torch.cat((empty, k_off)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,segments,heads", [
    ([1, 1, 1], [40, 3, 0], 2 ** 26 + 100, 1),
    ([500, 1, 70], [300, 9, 400], 2 ** 26 + 50, 2),  # two of them long
])
def test_more_segments_than_a_launch_has_workgroups(lq, lk, segments, heads):
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    host, q_off, k_off = _tail(lq, lk, segments, heads, 16, torch.float32)
    r = oracle.segment_attention(*host[:3], *host[4:], causal=True, gout=host[3])
    b = bounds(r, torch.float32)
    q, k, v, g = (x.cuda() for x in host[:4])
    out, saved = segment_attention_forward(q, k, v, q_off, k_off, causal=True)
    compare(out, r["out"], b["out"], "out")
    for name, x in zip(("gq", "gk", "gv"), segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off, causal=True)):
        compare(x, r[name], b[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_more_tiles_than_a_launch_has_workgroups(dtype, causal):
    """2^22 segments of one row each, whose output is their value and the gradient of that the output's, and one of 300 rows:
    above 2^24 workgroups of 256. Bounds as in test_attention.py, for scores with absolute sums below 64."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    ones, heads, dim = 2 ** 22 - 1, 4, 8
    host = make([300], [300], heads, heads, dim, dtype)
    off = torch.cat((torch.arange(ones + 1), torch.tensor([ones + 300]))).cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda x: torch.cat((torch.randn(ones, heads, dim, generator=gen, device="cuda").to(dtype), x.cuda()))  # noqa: E731
    q, k, v, g = (rows(x) for x in host[:4])
    r = oracle.segment_attention(*host[:3], *host[4:], causal=causal, gout=host[3])
    b = bounds(r, dtype)
    out, saved = segment_attention_forward(q, k, v, off, causal=causal)
    bound = lambda x: (2.0 * (16.0 * 2.0 ** -24 * 64.0 + 2.0 ** -20) + 1.01 * U[dtype]) * x.float().abs() + 1e-30  # noqa: E731
    assert bool(((out[:ones].float() - v[:ones].float()).abs() <= bound(v[:ones])).all())
    compare(out[ones:], r["out"], b["out"], "out")
    gq, gk, gv = segment_attention_vjp(g, q, k, v, out, saved, off, causal=causal)
    assert bool(((gv[:ones].float() - g[:ones].float()).abs() <= bound(g[:ones])).all())
    for name, x in zip(("gq", "gk", "gv"), (gq, gk, gv)):
        compare(x[ones:], r[name], b[name], name)


@pytest.mark.gpu
def test_more_deltas_than_a_launch_has_workgroups():
    """2^28 rows of a head, nearly all before the first segment: 16 of them a workgroup."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    heads, rows = 32, 2 ** 23 + 700
    host = make([200, 100], [200, 100], heads, heads, 8, torch.bfloat16)
    r = oracle.segment_attention(*host[:3], *host[4:], gout=host[3])
    b = bounds(r, torch.bfloat16)
    wide = lambda x: torch.cat((torch.zeros(rows - 300, heads, 8, dtype=x.dtype, device="cuda"), x.cuda()))  # noqa: E731
    q, g, k, v = wide(host[0]), wide(host[3]), host[1].cuda(), host[2].cuda()
    q_off, k_off = host[4].cuda() + rows - 300, host[5].cuda()
    out, saved = segment_attention_forward(q, k, v, q_off, k_off)
    gq, gk, gv = segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off)
    assert not out[:-300].any() and not gq[:-300].any()
    for name, x in (("out", out[-300:]), ("gq", gq[-300:]), ("gk", gk), ("gv", gv)):
        compare(x, r[name], b[name], name)


@pytest.mark.gpu
def test_more_rows_to_turn_than_a_launch_has_workgroups():
    """2^27 tokens, eight a workgroup: one row of features for all, each turned by its own position's angles."""
    from fastmd_amd.ops.qk_norm import rotary, rotary_tables

    tokens, dim = 2 ** 27 + 5, 136  # above 128 columns a row takes 32 lanes
    x = torch.randn(1, 1, dim, generator=torch.Generator().manual_seed(1)).bfloat16().cuda().expand(tokens, 1, dim)
    cos, sin = rotary_tables(1000, 16, device="cuda")
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32) % 1000
    out = rotary(x, cos, sin, positions)
    want = rotary(x[:1000], cos, sin, positions[:1000])
    at = 0
    for part in out.split(1000 * 1000):
        assert torch.equal(part[:len(part) // 1000 * 1000].view(-1, 1000, dim), want[:, 0].expand(len(part) // 1000, 1000, dim))
        at += len(part)
    assert at == tokens and torch.equal(out[-(tokens % 1000):], want[:tokens % 1000])


@pytest.mark.gpu
def test_too_many_tiles_are_refused():
    from fastmd_amd.ops.attention import segment_attention

    q = torch.zeros(2, 32, 8, device="cuda")
    off = torch.zeros(1, dtype=torch.int64, device="cuda").expand(2 ** 26 + 1)
    with pytest.raises(ValueError, match="2\\^31 tiles"):
        segment_attention(q, q, q, off)


def test_entry_point_refuses_too_many_tiles():
    from fastmd_amd import _abi

    assert _abi.load().fmd_segment_attention(0, 16, 256, 8, 16, 256, 8, 16, 256, 8, 16, 16, 2, 2, 2 ** 26, 32, 32, 8, 0, 1.0, 1,
                                             16, None, None, None, None, None) == 10001
