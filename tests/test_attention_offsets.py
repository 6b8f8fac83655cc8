"""(g) The tile search of segment attention on the host, and calls whose offsets do not ascend."""
import pytest
import torch

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
  for (int trial = 0; trial < 3000; ++trial) {
    const bool ascend = trial % 2;
    const int n = 1 + (int)pick(trial % 7 ? 8 : 300), group = 1 + (int)pick(4), bm = 32 << pick(3);
    const int64_t rows = pick(700);
    std::vector<int64_t> off(n + 1);
    for (auto& o : off) o = pick(rows + 60) - 30;
    if (ascend)
      for (int i = 1; i <= n; ++i)
        if (off[i] < off[i - 1]) off[i] = off[i - 1];
    std::vector<int> seen(rows * group, 0);
    for (int64_t t = 0; t < rows * group / bm + n + 2; ++t) {
      int64_t first = -1;
      const int s = attn_find(off.data(), n, rows, group, bm, t, &first, HostLanes());
      if (s < 0 || s > n + 1 || first < 0) return std::printf("trial %d, tile %lld: segment %d, row %lld", trial, (long long)t, s, (long long)first), 0;
      const int64_t q0 = attn_start(off.data(), n, rows, s);
      int64_t nq = (attn_start(off.data(), n, rows, s + 1) - q0) * group;
      if (nq < 0) nq = 0;
      for (int64_t r = first; r < nq && r < first + bm; ++r) {
        if (q0 * group + r >= rows * group) return std::printf("trial %d: row outside", trial), 0;
        ++seen[q0 * group + r];
      }
    }
    if (ascend)
      for (int x : seen)
        if (x != 1) return std::printf("trial %d: a row in %d tiles", trial, x), 0;
  }
  std::printf("ok");
}
"""


def test_every_row_is_in_one_tile_and_no_tile_outside(tmp_path):
    """Ascending offsets (clamped ones, empty segments, rows outside all): each packed row in one tile. Any others: every tile
    within the buffer."""
    assert run_host(tmp_path, HOST) == "ok"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offsets", [[0, 300, 100, 400], [400, 0, 400], [399, -5, 700, 2, 400], [400, 300, 200, 0]])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 8)])
def test_descending_offsets_stay_in_bounds(heads, kv_heads, offsets, dtype):
    """Such a call ends, and the inputs keep their values (which rows it computes is open)."""
    from fastmd_amd.ops.attention import segment_attention_forward, segment_attention_vjp

    gen = torch.Generator().manual_seed(2)
    rand = lambda h: torch.randn(400, h, 64, generator=gen).to(dtype).cuda()  # noqa: E731
    q, g, k, v = rand(heads), rand(heads), rand(kv_heads), rand(kv_heads)
    kept = [x.clone() for x in (q, g, k, v)]
    off = torch.tensor(offsets, device="cuda")
    for causal in (False, True):
        out, saved = segment_attention_forward(q, k, v, off, causal=causal)
        segment_attention_vjp(g, q, k, v, out, saved, off, causal=causal)
    torch.cuda.synchronize()
    for x, y in zip((q, g, k, v), kept):
        assert torch.equal(x, y)
