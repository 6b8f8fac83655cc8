// Which segment a tile of rows belongs to, from the segments' offsets. Host code too, with the wave's lanes taken in turn.
//
// The kernels see segments + 2 of them: the rows before the first offset and after the last one (a fixed-capacity
// buffer's unused rows) are segments of their own without keys, or without queries.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

// start of extended segment i in 0 .. n + 2, with every offset clamped into the buffer
__host__ __device__ __forceinline__ int64_t attn_start(const int64_t* off, int n, int64_t rows, int i) {
  if (i == 0) return 0;
  if (i == n + 2) return rows;
  const int64_t o = off[i - 1];
  return o < 0 ? 0 : o > rows ? rows : o;
}

// The number of lanes of a wave that a condition holds for.
struct WaveLanes {
  template <typename At>
  __device__ __forceinline__ int operator()(const At& at) const { return __popcll(__ballot(at((int)(threadIdx.x & 63)))); }
};

// The last i of 0 .. count - 1 with number(i) <= t, for ascending numbers from 0 on. It probes 64 places at a time.
template <typename Number, typename Lanes>
__host__ __device__ __forceinline__ int attn_last(int count, int64_t t, const Number& number, const Lanes& lanes) {
  int lo = 0;
  while (count > 1) {
    const int step = (count + 63) >> 6;
    const int hits = lanes([&](int lane) { return lane * step < count && number(lo + lane * step) <= t; });
    const int adv = (hits > 0 ? hits - 1 : 0) * step;
    lo += adv;
    count = count - adv < step ? count - adv : step;
  }
  return lo;
}

// The tile of `bm` packed rows (rows * group of them) with number t: extended segment i owns the numbers from
// floor(start(i) * group / bm) + i on, at least as many as it has tiles, so no table of tiles is needed and the grid
// (rows * group / bm + segments + 2) is known without reading the offsets.
// Returns the extended segment and the tile's first packed row in it; a number without a tile has first row >= rows, and so has
// one before its segment's first, which the search ends on only where offsets descend (the caller's error: which rows
// such a call computes is open, but it stays within the buffers).
template <typename Lanes>
__host__ __device__ __forceinline__ int attn_find(const int64_t* off, int n, int64_t rows, int group, int bm, int64_t t, int64_t* first,
                                                  const Lanes& lanes) {
  const auto number = [&](int i) { return attn_start(off, n, rows, i) * group / bm + i; };
  const int i = attn_last(n + 2, t, number, lanes);
  const int64_t tile = t - number(i);
  *first = tile < 0 ? INT64_MAX : tile * bm;
  return i;
}

// The row kernels give a segment to one wave. One of kLongQueries queries or kLongKeys keys and more, whatever the mean over all
// segments is, is dealt out over workgroups instead: its share of numbers from floor(q / kLongQueries) + floor(k / kLongKeys) on,
// q and k its first rows, at least one. The grid (tq / kLongQueries + tk / kLongKeys) is known without reading the offsets. Nearly always
// they find no such segment: us of forward, VJP without them and with, and with four times as many for the queries: 10 000 segments of 18 keys,
// 4 heads of 32, bf16 20, 34; 20, 34; 22, 36; 100 000 of 20 keys 191, 378; 208, 392; 232, 425, fp32 380, 850; 389, 865; 412, 895. (Between the
// rows' workgroups instead of after them they shift those from one CU to another: 1 024 segments of 500 keys, VJP 225; 226; 315.)
constexpr int kLongQueries = 32, kLongKeys = 1024;

__host__ __device__ __forceinline__ bool attn_long(int nq, int nk) { return nq >= kLongQueries || nk >= kLongKeys; }
__host__ __device__ __forceinline__ int64_t attn_long_numbers(int64_t tq, int64_t tk) { return tq / kLongQueries + tk / kLongKeys; }

// The extended segment of number t, and which of its parts the number is (part >= parts: none).
template <typename Lanes>
__host__ __device__ __forceinline__ int attn_share(const int64_t* q_off, const int64_t* k_off, int n, int64_t tq, int64_t tk, int64_t t,
                                                   int64_t* part, int64_t* parts, const Lanes& lanes) {
  const auto number = [&](int i) { return attn_long_numbers(attn_start(q_off, n, tq, i), attn_start(k_off, n, tk, i)); };
  const int i = attn_last(n + 2, t, number, lanes);
  *part = t - number(i);
  *parts = *part < 0 ? 0 : number(i + 1) - number(i);
  if (*part < 0) *part = 0;
  return i;
}
