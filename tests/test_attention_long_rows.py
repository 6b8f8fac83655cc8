"""(g) Segment attention of about one query per segment where some segments are long all the same: slots mostly empty, one
context far longer than the rest. Their work is dealt out over workgroups, not left to one wave."""
import pytest
import torch

from test_attention import TYPES, check, make
from test_host_math import run_host

HOST = r"""
#include <hip/hip_runtime.h>
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "attention_find.h"
struct HostLanes {
  template <typename At>
  int operator()(const At& at) const {
    int n = 0;
    for (int lane = 0; lane < 64; ++lane) n += at(lane);
    return n;
  }
};
static int64_t pick(int64_t n) { return n > 0 ? rand() % n : 0; }
int main() {
  for (int trial = 0; trial < 2000; ++trial) {
    const bool ascend = trial % 4 != 0;
    const int n = 1 + (int)pick(trial % 7 ? 20 : 300);
    std::vector<int64_t> q(n + 1), k(n + 1);
    int64_t tq = pick(5), tk = pick(900);
    for (int i = 0; i <= n; ++i) {
      q[i] = tq;
      k[i] = tk;
      tq += pick(3) ? pick(2) : pick(60);
      tk += pick(5) ? pick(30) : pick(5000);
    }
    if (!ascend)
      for (int i = 0; i < 3; ++i) std::swap(q[pick(n + 1)], q[pick(n + 1)]), std::swap(k[pick(n + 1)], k[pick(n + 1)]);
    std::vector<std::vector<int>> seen(n + 2);
    std::vector<int64_t> all(n + 2, 0);
    for (int64_t t = 0; t < attn_long_numbers(tq, tk); ++t) {
      int64_t part = -1, parts = -1;
      const int i = attn_share(q.data(), k.data(), n, tq, tk, t, &part, &parts, HostLanes());
      if (i < 0 || i > n + 1 || part < 0) return std::printf("trial %d number %lld", trial, (long long)t), 0;
      if (part >= parts) continue;
      if (parts > attn_long_numbers(tq, tk)) return std::printf("trial %d: %lld parts", trial, (long long)parts), 0;
      all[i] = parts;
      seen[i].resize(parts);
      ++seen[i][part];
    }
    if (!ascend) continue;
    for (int i = 1; i <= n; ++i) {
      const int nq = (int)(q[i] - q[i - 1]), nk = (int)(k[i] - k[i - 1]);
      if (!attn_long(nq, nk)) continue;
      if (all[i] < nq / kLongQueries || all[i] < nk / kLongKeys || all[i] < 1)
        return std::printf("trial %d: %lld parts of %d queries, %d keys", trial, (long long)all[i], nq, nk), 0;
      for (int x : seen[i])
        if (x != 1) return std::printf("trial %d: a part %d times", trial, x), 0;
    }
  }
  std::printf("ok");
}
"""


def test_parts_of_long_segments(tmp_path):
    """Every part of a long segment has one number, as many parts as its queries and keys ask for; offsets that descend
    lead nowhere outside."""
    assert run_host(tmp_path, HOST) == "ok"


def _slots(count, lengths):
    gen = torch.Generator().manual_seed(count)
    lq = torch.randint(0, 2, (count,), generator=gen).tolist()
    lk = torch.randint(0, 20, (count,), generator=gen).tolist()
    for slot, (nq, nk) in lengths.items():
        lq[slot], lk[slot] = nq, nk
    while sum(lq) > count:
        lq[lq.index(1)] = 0
    return lq, lk


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 32), (3, 1, 24), (4, 2, 128), (4, 1, 64), (20, 10, 72)])
def test_long_segments_among_short_ones(heads, kv_heads, dim, dtype, causal):
    lq, lk = _slots(600, {0: (1, 1024), 7: (31, 1023), 8: (32, 30), 100: (90, 170), 101: (33, 0), 102: (40, 5), 598: (2, 2500), 599: (0, 1500)})
    assert sum(lq) <= 600 and sum(lk) <= 32 * 600  # few enough for the row kernels, of any group
    q, k, v, g, q_off, k_off = make(lq, lk, heads, kv_heads, dim, dtype, before=4, after=70, seed=dim)
    check(q, k, v, g, q_off, k_off, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_one_long_sequence_among_empty_slots_is_not_one_waves_work(dtype):
    """2 048 slots, one of 1 500 queries over 1 500 keys: 2 250 000 pairs per head. A wave takes some 10^6 steps for each direction,
    about a second; dealt out the pair of calls takes a few milliseconds. The bound lies a factor of ten from both."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    lengths = [1500 if s == 5 else 0 for s in range(2048)]
    q, k, v, g, off, _ = (x.cuda() for x in make(lengths, lengths, 4, 4, 32, dtype))

    def run():
        out, saved = segment_attention_forward(q, k, v, off)
        return segment_attention_vjp(g, q, k, v, out, saved, off)

    run()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    run()
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 100.0


@pytest.mark.gpu
def test_long_segments_repeat_bitwise():
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    lq, lk = _slots(300, {100: (150, 170), 298: (2, 2500)})
    q, k, v, g, q_off, k_off = (x.cuda() for x in make(lq, lk, 4, 2, 32, torch.float32))

    def run():
        out, saved = segment_attention_forward(q, k, v, q_off, k_off)
        return (out, *segment_attention_vjp(g, q, k, v, out, saved, q_off, k_off))

    for a, b in zip(run(), run()):
        assert torch.equal(a, b)
