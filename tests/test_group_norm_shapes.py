"""(h) What the host decides for the norm over groups of channels, and parameters that do not start on whole vectors."""
import pytest
import torch

from test_group_norm import TYPES, check, make, ragged
from test_host_math import run_host

HOST = r"""
#include <cstdio>
#include "group_norm_shapes.h"
static GnArgs call(int64_t rows, int channels, int groups, int segments, uintptr_t x, uintptr_t weight, uintptr_t bias, uintptr_t y) {
  static const int64_t off = 0;
  GnArgs a{};
  a.rows = rows, a.channels = channels, a.groups = groups, a.width = channels / groups, a.segments = segments;
  a.x = reinterpret_cast<void*>(x), a.y = reinterpret_cast<void*>(y);
  a.weight = reinterpret_cast<void*>(weight), a.bias = reinterpret_cast<void*>(bias);
  a.x_ld = a.g_ld = channels, a.off = segments ? &off : nullptr;
  return a;
}
int main() {
  const uintptr_t at = 1 << 20;
  for (int size = 2; size <= 4; size += 2)
    for (int64_t shift = 0; shift <= 16; shift += size)
      for (int which = 0; which < 3; ++which) {
        const uintptr_t p[3] = {at + (which == 0 ? shift : 0), at + (which == 1 ? shift : 0), at + (which == 2 ? shift : 0)};
        GnArgs a = call(700, 128, 8, 3, at, p[0], p[1], p[2]);
        const TileShape s = tile_shape(a, size, false);
        set_tiles(a, s, size);
        const int64_t bytes = s.v * size;
        if (p[2] % bytes) return std::printf("results stored across vectors"), 0;
        if (a.params_wide && (p[0] % bytes || p[1] % bytes)) return std::printf("parameters read across vectors"), 0;
        if (shift % 16 == 0 && !(a.params_wide && bytes == 16)) return std::printf("narrow without need"), 0;
      }
  GnArgs a = call(700, 128, 8, 3, at, 0, 0, at);
  set_tiles(a, tile_shape(a, 2, false), 2);
  std::printf(a.params_wide ? "ok" : "no parameters: nothing to read");
}
"""


def test_vectors_lie_whole_in_memory(tmp_path):
    assert run_host(tmp_path, HOST) == "ok"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,groups,lengths", [(128, 8, [40, 60]), (320, 32, [700, 0, 90]), (2048, 2, [9, 30]), (48, 3, [3000])])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_parameters_from_within_a_packed_one(shift, channels, groups, lengths, dtype):
    """Contiguous, but not on whole vectors, beside features that are."""
    x, w, b, gy = make(sum(lengths), channels, dtype)

    class Shifted:  # what check() puts on the GPU
        def __init__(self, t, n):
            self.t, self.n = t, n

        def cuda(self):
            pack = torch.zeros(self.t.numel() + self.n, dtype=self.t.dtype, device="cuda")
            pack[self.n:] = self.t.cuda()
            return pack[self.n:]

        def double(self):
            return self.t.double()

    check(x, groups, Shifted(w, shift), Shifted(b, shift), gy, ragged(lengths), "silu")
    check(x, groups, w, Shifted(b, shift), gy, ragged(lengths), "silu")
