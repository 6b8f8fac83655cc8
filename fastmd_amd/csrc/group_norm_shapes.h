// Of the norm over groups of channels, what the host decides: vectors, tiles, workgroups. Without kernels: a host test includes it.
#pragma once

#include <cstdint>

constexpr int kThreads = 256;
constexpr int kTileValues = 64;     // of a thread's registers: the forward pass's rows of a tile
constexpr int kBackParts = 8;       // the backward pass's: half as many values of both inputs, up to eight times over (262 144 rows of 128,
                                    // bf16: first read 56 us with one part, 43 with four, 42 with eight; second 43, 39, 39)
constexpr int64_t kFewTiles = 1024; // tiles are made smaller below this number of them

struct GnArgs {
  const void *x, *g;  // rows [rows, channels], row strides x_ld, g_ld; g: gradient of y
  int64_t x_ld, g_ld;
  const void *weight, *bias;  // [channels], or null: ones, zeros
  int32_t params_wide;        // segments: both start on whole vectors
  const int64_t* off;         // [segments + 1]
  int64_t rows;
  int32_t segments, channels, groups, width, act;
  float eps;
  void *y, *gx;          // contiguous
  float *mean, *inverse;  // [rows or segments, groups]
  float *part;           // scratch (see the kernels)
  int64_t again;         // workgroups of the second read by the numbers of the first (a multiple of 8), or 0
  int32_t merge;         // whether gn_merge_kernel merges the sums of segments of many tiles
  int32_t chunk;         // channels of a workgroup's share (whole groups)
  int32_t tile_rows, tx;  // rows of a tile, vectors of a row of the share
  int32_t part_rows;      // backward: rows that are in registers at once
  int32_t lanes;         // rows by themselves: lanes of a group
  int32_t blocks;        // of rows, in x
  uint32_t block0;
};

// Each workgroup of the second read merges the sums of its segment's tiles itself where all tiles' together are few (kMergeValues);
// otherwise those of a segment of more than kMergeTiles tiles are merged once, by gn_merge_kernel: 33 tiles of 8 groups each 48 us with
// a launch for it, 47 without (16 875 rows of 128, float32, with VJP); 85 tiles of 32 groups 80 us by each workgroup, 38 by the launch.
constexpr int kMergeTiles = 16;
constexpr int64_t kMergeValues = 8192;

inline bool aligned(const void* p, int64_t ld, int64_t bytes, int size) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && ld * size % bytes == 0;
}

// the widest vector, of up to 16 bytes, of which `unit` channels are whole ones and on which the rows of what is read and written start
inline int vector_of(const GnArgs& a, int size, int64_t unit) {
  for (int v = 16 / size; v > 1; v >>= 1)
    if (unit % v == 0 && a.channels % v == 0 && aligned(a.x, a.x_ld, v * size, size) && (!a.g || aligned(a.g, a.g_ld, v * size, size)) &&
        aligned(a.y, 0, v * size, size) && aligned(a.gx, 0, v * size, size))
      return v;
  return 1;
}

// Rows by themselves: lanes of a group and vectors of a lane
struct RowShape {
  int v, nv, lanes;
  bool wide;
};

inline RowShape row_shape(const GnArgs& a, int size) {
  RowShape s{};
  s.v = vector_of(a, size, a.width);
  const int vectors = a.width / s.v;
  s.wide = vectors > 256;
  if (s.wide) {
    s.lanes = kThreads;
    s.nv = (vectors + kThreads - 1) / kThreads;
  } else {
    for (s.lanes = 1; s.lanes < 64 && s.lanes < vectors; s.lanes *= 2) {}
    s.nv = (vectors + s.lanes - 1) / s.lanes;
  }
  return s;
}

// rows and groups of a workgroup, as GnUnits
inline int row_groups(const GnArgs& a, const RowShape& s) {
  const int n = kThreads / s.lanes;
  return a.groups < n ? a.groups : n;
}

// The backward pass's workgroups: each walks rows, and its channels' sums are a row of the last step's input
constexpr int64_t kRowBlocks = 512;

inline int64_t row_blocks(const GnArgs& a, const RowShape& s) {
  const int at_once = row_groups(a, s), rows = kThreads / s.lanes / at_once;
  const int64_t all = (a.rows + rows - 1) / rows;
  return all < kRowBlocks ? all : kRowBlocks;
}

// Segments: a workgroup's share of the channels, whole groups of them; its tile's rows
struct TileShape {
  int v, nv, nr, chunk, tx, rows, part_rows, chunks, lds;
};

inline TileShape tile_shape(const GnArgs& a, int size, bool back) {
  TileShape s{};
  for (s.v = vector_of(a, size, a.channels);; s.v >>= 1) {
    const int most = kThreads * s.v;
    s.chunk = a.channels;
    if (a.channels > most) {
      int groups = most / a.width;  // the most groups that a row of threads takes, as whole vectors
      while (groups > 1 && groups * a.width % s.v) --groups;
      s.chunk = (groups > 0 ? groups : 1) * a.width;
    }
    if (s.v == 1 || s.chunk % s.v == 0) break;
  }
  s.tx = s.chunk / s.v;
  s.nv = s.tx > kThreads ? (s.tx + kThreads - 1) / kThreads : 1;
  const int most = 32 / s.v;  // registers of the wide forms: 8 192 channels of a group at most
  if (s.nv > 1) s.nv = s.nv <= 4 ? 4 : s.nv <= most ? most : -1;
  const int rows = s.nv > 1 ? 1 : kThreads / s.tx;
  // forward: up to 64 values of a thread, all in registers; backward: 32 of each input at a time, eight times over. Fewer where the tiles
  // would not fill the card.
  s.nr = s.nv > 1 ? (s.v * s.nv < 16 ? 16 / (s.v * s.nv) * 2 : 2) : s.v == 1 ? 32 : kTileValues / s.v;
  int passes = back ? kBackParts : 1;
  if (back && s.nv == 1) s.nr /= 2;
  while (passes > 1 && a.rows / (passes * s.nr * rows) < kFewTiles) passes /= 2;
  if (s.nv == 1)
    for (int i = back ? 1 : 0; i < 2 && a.rows / (s.nr * rows) < kFewTiles; ++i) s.nr /= 2;
  s.part_rows = s.nr * rows;
  s.rows = passes * s.part_rows;
  s.chunks = (a.channels + s.chunk - 1) / s.chunk;
  s.lds = ((back ? 2 : 1) * rows * s.chunk + 2 * (s.chunk / a.width)) * 4;
  return s;
}

inline int64_t tile_count(const GnArgs& a, const TileShape& s) { return a.rows / s.rows + a.segments + 2; }
inline int64_t second_count(const GnArgs& a, const TileShape& s) { return a.again ? a.again : 2 * a.rows / s.rows + 1; }

inline void set_tiles(GnArgs& a, const TileShape& s, int size) {
  a.chunk = s.chunk;
  a.tx = s.tx;
  a.tile_rows = s.rows;
  a.part_rows = s.part_rows;
  a.params_wide = aligned(a.weight, 0, s.v * size, size) && aligned(a.bias, 0, s.v * size, size);
  a.again = a.segments <= a.rows / s.rows ? (a.rows / s.rows + a.segments + 2 + 7) / 8 * 8 : 0;
  a.merge = a.rows / s.rows * a.groups > kMergeValues && a.rows > (int64_t)kMergeTiles * s.rows;
}
