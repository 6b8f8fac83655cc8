"""(h) The norm over groups of channels where calls are large enough for what small ones do not run: tiles of several parts of rows in the
VJP, the sums of many tiles merged by a launch of their own, and a second round of rows by themselves. A host test holds each size
to what it is listed for."""
import pytest
import torch

from oracle import blocks as oracle
from test_group_norm import TYPES, make, ragged
from test_host_math import run_host

F32, BF16 = TYPES

# type, channels, groups, lengths, lead, spare, parts of rows of a tile in the VJP
PARTS = [
    (F32, 128, 8, [70001, 0, 129, 1, 127, 128, 64777], 200, 333, 2),
    (BF16, 128, 32, [70001, 0, 129, 16, 127, 128, 64777], 200, 333, 2),
    (F32, 35, 5, [300001, 449, 448, 447, 170003], 500, 700, 4),
    (BF16, 35, 7, [300001, 449, 448, 447, 170003], 500, 700, 4),
    (F32, 257, 1, [40001, 65, 0, 64, 63, 26003], 90, 75, 8),
    (BF16, 1031, 1, [9001, 17, 0, 16, 15, 8003], 20, 35, 8),
    (BF16, 4100, 1, [9001, 17, 0, 16, 15, 8003], 20, 35, 8),
]
# type, channels, groups, lengths; the merge by segments, or by numbers where there are more segments than could be long
MERGED = [
    (F32, 64, 32, [30000, 0, 19001, 500], False),
    (BF16, 64, 32, [30000, 0, 19001, 500], False),
    (F32, 64, 32, [17] * 60 + [30000] + [0, 21] * 40 + [9001] + [1500] * 3, True),
    (BF16, 64, 32, [17] * 60 + [30000] + [0, 21] * 40 + [9001] + [1500] * 3, True),
    (BF16, 99, 33, [31] * 90 + [40007, 0, 20001] + [16] * 60, True),
]
# type, channels, groups, rows: tiles of more rows than small calls have, in vectors of each width
TILES = [(F32, 128, 8, 68001), (F32, 130, 5, 66003), (F32, 130, 26, 131002), (BF16, 132, 3, 66003), (BF16, 132, 12, 132001), (BF16, 130, 13, 66001),
         (BF16, 128, 4, 70003)]
# type, channels, rows of one group: vectors of a lane, in vectors of each width
ROWS = [(dtype, channels, 1) for dtype in TYPES for channels in (63, 99, 255, 66, 130, 258, 300, 400, 1000, 1020, 520, 2040)]
# type, channels, groups, rows: more workgroups of rows than there are in a launch
ROUNDS = [
    (F32, 1024, 1, 2101), (BF16, 1024, 1, 2101), (F32, 8192, 1, 601), (BF16, 8190, 1, 601), (F32, 2048, 64, 700), (BF16, 999, 3, 1900),
    (BF16, 512, 8, 3000),
]


def shapes(tmp_path, calls):
    """[(parts of rows, rows of a part, whether merged: forward and VJP, by numbers: both, workgroups of rows by themselves, and their rows)]"""
    body = "\n".join(f"  show({rows}, {channels}, {groups}, {segments}, {2 if dtype == BF16 else 4});"
                     for dtype, channels, groups, rows, segments in calls)
    out = run_host(tmp_path, r"""
#include <cstdio>
#include "group_norm_shapes.h"
static void show(int64_t rows, int channels, int groups, int segments, int size) {
  static const int64_t off = 0;
  GnArgs a{};
  a.rows = rows, a.channels = channels, a.groups = groups, a.width = channels / groups, a.segments = segments;
  a.x_ld = a.g_ld = channels, a.off = segments ? &off : nullptr;
  const TileShape f = tile_shape(a, size, false), b = tile_shape(a, size, true);
  GnArgs fa = a, ba = a;
  set_tiles(fa, f, size);
  set_tiles(ba, b, size);
  const RowShape r = row_shape(a, size);
  std::printf("%d %d %d %d %d %d %d %d\n", b.rows / b.part_rows, b.part_rows, fa.merge, ba.merge, rows / (kMergeTiles * f.rows) < segments,
              rows / (kMergeTiles * b.rows) < segments, (int)row_blocks(a, r), kThreads / r.lanes / row_groups(a, r));
}
int main() {
""" + body + "\n}\n")
    return [tuple(int(n) for n in line.split()) for line in out.splitlines()]


def test_the_sizes_are_what_they_are_listed_for(tmp_path):
    calls = [(d, c, g, sum(n) + lead + spare, len(n)) for d, c, g, n, lead, spare, _ in PARTS]
    for (_, _, _, lengths, lead, spare, parts), (got, part, *_) in zip(PARTS, shapes(tmp_path, calls)):
        assert got == parts and min(lead, spare) > part
        assert part * parts + 1 in lengths and part * parts in lengths and part * parts - 1 in lengths  # about a tile
    calls = [(d, c, g, sum(n), len(n)) for d, c, g, n, _ in MERGED]
    for (_, _, _, lengths, by_number), (_, _, forward, back, number, back_number, *_) in zip(MERGED, shapes(tmp_path, calls)):
        assert forward and back and (number, back_number) == (by_number, by_number)
    for (_, _, _, rows), (*_, workgroups, each) in zip(ROUNDS, shapes(tmp_path, [(d, c, g, rows, 0) for d, c, g, rows in ROUNDS])):
        assert workgroups * each < rows


def check(dtype, channels, groups, rows, offsets, activation="silu", lead=0, spare=0):
    from fastmd_amd.ops.group_norm import group_norm_forward, group_norm_vjp

    x, w, b, gy = make(rows, channels, dtype)
    x[:lead] = float("nan")
    x[rows - spare:] = float("inf")
    want = oracle.group_norm(x, groups, w, b, offsets, name=activation, gy=gy)
    x, w, b, gy = (t.cuda() for t in (x, w, b, gy))
    off = None if offsets is None else offsets.cuda()
    y, saved = group_norm_forward(x, groups, w, b, offsets=off, activation=activation)
    got = (y, *group_norm_vjp(gy, x, groups, w, b, saved, offsets=off, activation=activation))
    alone = group_norm_vjp(gy, x, groups, w, b, saved, offsets=off, activation=activation, need_weights=False)
    assert torch.equal(alone[0], got[1])
    for name, t, (value, bound) in zip(("y", "gx", "gw", "gb"), got, want):
        oracle.near(t, value, bound, name)
    for t in got[:2]:
        assert not t[:lead].any() and not t[rows - spare:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,channels,groups,lengths,lead,spare,parts", PARTS)
def test_several_parts_of_rows_a_tile(dtype, channels, groups, lengths, lead, spare, parts):
    check(dtype, channels, groups, sum(lengths) + lead + spare, ragged(lengths, lead), lead=lead, spare=spare)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,channels,groups,rows", TILES)
def test_tiles_of_many_rows(dtype, channels, groups, rows):
    check(dtype, channels, groups, rows, ragged([rows // 2 - 50, 300, rows - rows // 2 - 250]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,channels,groups", ROWS)
def test_vectors_of_a_lane(dtype, channels, groups):
    check(dtype, channels, groups, 37, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,channels,groups,lengths,by_number", MERGED)
def test_sums_of_many_tiles_merged_by_a_launch(dtype, channels, groups, lengths, by_number):
    check(dtype, channels, groups, sum(lengths), ragged(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,channels,groups,rows", ROUNDS)
def test_rows_past_the_first_round(dtype, channels, groups, rows):
    check(dtype, channels, groups, rows, None)
