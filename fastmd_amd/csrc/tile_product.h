// Products out[m, n] = sum_k n_op[n, k] m_op[m, k] on the matrix cores, with the result's own use as an epilogue: what the
// gated feed-forward block and the 8-bit product are made of.
//
// Both operands of a slice of K are copied straight from global memory into LDS (no register stage), into two places in turn: while
// the matrix instructions run on one slice, the next is on its way. An operand is stored along K (its rows are rows of the product, K
// contiguous) or across it (its rows are K, as a weight is in the products of the backward pass); the second kind is
// transposed by the LDS reads (ds_read_b64_tr_b16), never in memory. The n operand is the matrix instruction's first: a
// lane's four consecutive results then lie side by side in a row of the output.
//
// float32 operands come as three bf16 planes (x3.h); their six plane products follow each other along K, the small ones
// first, in one accumulator: K is six times as long, the kernel is the same. Likewise an operand of two planes (16 bits) against one of bf16.
#pragma once

#include "common.h"
#include "x3.h"

typedef int tp_i32x4 __attribute__((ext_vector_type(4)));
typedef int tp_i32x16 __attribute__((ext_vector_type(16)));
typedef short tp_s16x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kTpMostLd = int64_t(1) << 23;  // bytes: a lane's offset in the 256 rows of a tile fits 32 bits

// base: of each part of K (a sum of two products), or, for a gated product, of the two matrices whose rows share a tile
struct TpOperand {
  const char* base[2];
  int64_t ld, plane;  // bytes from a stored row to the next, and from a plane to the next
};

// The products of planes, in their order along K: two bits each, the plane of n and that of m
struct TpPairs {
  int32_t count;
  uint32_t n, m;
};
constexpr TpPairs kTpPlain{1, 0, 0}, kTpThree{6, 0x124, 0x046};  // of three planes each: (0,2) (1,1) (2,0) (0,1) (1,0) (0,0)
constexpr TpPairs kTpTwoN{2, 1, 0}, kTpTwoM{2, 0, 1};            // n, or m, of two planes

struct TpProblem {
  TpOperand n, m;
  int64_t rows_n, rows_m, k;  // of one part
  int32_t parts;              // of K
  TpPairs pairs;
  int32_t tiles_n, tiles_m, first;  // tiles, and the number of the first one
};

constexpr int kTpProblems = 3;

// Tiles [0, full) are whole; each of the others is shared by `splits` workgroups that take a part of its K each and leave their
// sums in `partial`, [tile, split, value, thread] in units of four, for tile_join_kernel.
struct TpArgs {
  TpProblem p[kTpProblems];
  int32_t count, tiles, full, splits;
  void* partial;
};

typedef uint32_t tp_u32x4 __attribute__((ext_vector_type(4)));

constexpr int tp_wait(int vm, int lgkm) { return (vm & 15) | (7 << 4) | (lgkm << 8); }  // s_waitcnt vmcnt(vm) lgkmcnt(lgkm)

struct TpBf16 {
  typedef fmd_f32x16 Acc;
  static constexpr int SIZE = 2;
  __device__ static __forceinline__ Acc mma(tp_i32x4 a, tp_i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(fmd_bf16x8, a), __builtin_bit_cast(fmd_bf16x8, b), c, 0, 0, 0);
  }
};
struct TpInt8 {
  typedef tp_i32x16 Acc;
  static constexpr int SIZE = 1;
  __device__ static __forceinline__ Acc mma(tp_i32x4 a, tp_i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};

// One operand's rows in LDS: ROWS rows of the product, SLICE bytes of K each (along), or SLICE / 2 rows of K (across). 16-byte
// chunks are permuted so that neither kind of read meets one of the 64 banks twice: sixteen consecutive rows' same chunk (along), or
// four chunks of four consecutive rows of K (across).
constexpr int kTpSlice = 128;  // bytes of K in a slice
constexpr int kTpSteps = kTpSlice / 32, kTpRow = kTpSlice / 16;  // steps of the matrix instructions, chunks of a row
// Two places: four of half a slice each (four chunks a row: half lines of memory, twice the barriers) took 202 us for 8 192 x 2 048 over
// K = 5 504, bf16, against 186, and 480 us against 296 in tiles of 64 x 64.
constexpr int kTpPlaces = 2;

template <int ROWS, bool ACROSS_, bool GATED, int THREADS>
struct TpStage {
  static constexpr bool ACROSS = ACROSS_;
  static constexpr int BYTES = ROWS * kTpSlice, LOADS = BYTES / 16 / THREADS;
  static constexpr int WIDTH = ROWS * 2, CHUNKS = ROWS / 8;  // across: bytes and chunks of a row of K
  static_assert(BYTES % (16 * THREADS) == 0, "whole passes");
  static_assert(!(ACROSS && GATED), "a gated product's weights lie along K");

  __device__ static __forceinline__ int swap_along(int row) { return (row & 7) ^ ((row >> 3) & 1); }
  __device__ static __forceinline__ int swap_across(int row) { return CHUNKS >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

  uint32_t off[LOADS];
  int k;  // bytes of K before this lane's (of its first copy)
  const char* at[GATED ? 2 : 1];
  int64_t step;

  // this thread's offsets for the tile whose first row is `row0` (below `rows`)
  __device__ __forceinline__ void place(const TpOperand& o, int64_t row0, int64_t rows, int wave, int lane) {
    step = ACROSS ? (kTpSlice / 2) * o.ld : kTpSlice;
    k = ACROSS ? lane / CHUNKS * 2 : ((lane % kTpRow) ^ swap_along(lane / kTpRow)) * 16;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int slot = (wave * LOADS + j) * 64 + lane;
      if (ACROSS) {
        const int row = slot / CHUNKS, chunk = (slot % CHUNKS) ^ swap_across(row);
        const int64_t last = ((rows + 7) & ~int64_t(7)) - 8 - row0;  // chunks past the rows: the last one again, never used
        off[j] = (uint32_t)(row * o.ld) + 2 * (uint32_t)(chunk * 8 < last ? chunk * 8 : last);
      } else {
        int row = slot / kTpRow;
        const int chunk = (slot % kTpRow) ^ swap_along(row);
        if (GATED && row >= ROWS / 2) row -= ROWS / 2;
        const int64_t last = rows - 1 - row0;
        off[j] = (uint32_t)((row < last ? row : last) * o.ld) + 16 * chunk;
      }
    }
  }

  // the copies start at slice `slice` of a part and plane
  __device__ __forceinline__ void begin(const TpOperand& o, int part, int plane, int64_t row0, int slice) {
    const int64_t from = plane * o.plane + slice * step + row0 * (ACROSS ? 2 : o.ld);
    if (GATED) {
      at[0] = o.base[0] + from;
      at[GATED ? 1 : 0] = o.base[1] + from;
    } else {
      at[0] = o.base[part] + from;
    }
  }

  // Copy j of the slice at `at` to LDS, 64 lanes' 16 bytes; of K `left` bytes are left, past them is zero (an offset past the
  // buffer's end). As an instruction: after the compiler's own form every read of LDS waits for all copies, those to other places
  // too. tile_product_kernel holds the waits.
  __device__ __forceinline__ void copy(uint32_t lds, int j, int left, int wave) const {
    const int n = wave * LOADS + j;
    const char* base = GATED && n * (64 / kTpRow) >= ROWS / 2 ? at[GATED ? 1 : 0] : at[0];
    const tp_u32x4 buffer = {(uint32_t)(uintptr_t)base, (uint32_t)((uintptr_t)base >> 32) & 0xffff, 0x80000000u, 0x00027000u};
    const int mine = ACROSS ? k : k ^ (16 * (n & 1)), rest = ACROSS ? left - n * (64 / CHUNKS) * 2 : left;
    const uint32_t from = mine < rest ? off[j] : 0xffffffffu;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds + n * 1024), "v"(from), "s"(buffer)
                 : "memory", "m0");
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int g = 0; g < (GATED ? 2 : 1); ++g) at[g] += step;
  }

  // a lane's place in the operand reads
  __device__ static __forceinline__ int lane_at(int lane) {
    const int h = lane >> 5;
    if (ACROSS) {
      const int row = 8 * h + ((lane & 15) >> 2);
      return row * WIDTH + ((((lane >> 4) & 1) * 32 + (lane & 3) * 8) ^ (swap_across(row) * 16));
    }
    const int row = lane & 31;
    return row * kTpSlice + ((h ^ swap_along(row)) << 4);
  }

  // operand of the 32 rows from `row` (a multiple of 32) over step kk of a slice: 16 bytes, from K 32 kk + 16 (lane / 32) bytes
  __device__ static __forceinline__ tp_i32x4 read(const char* lds, int at, int row, int kk) {
    if (ACROSS) {
      typedef __attribute__((address_space(3))) tp_s16x4* lds_ptr;
      const char* x = lds + kk * 16 * WIDTH + (at ^ (row * 2));
      const tp_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)x);
      const tp_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(x + 4 * WIDTH));
      return __builtin_bit_cast(tp_i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *reinterpret_cast<const tp_i32x4*>(lds + row * kTpSlice + (at ^ (kk << 5)));
  }
};

// WN x WM waves, each with NB x MB blocks of 32 x 32. A wave's n blocks are half in the tile's first half of n, half in the
// second: of a gated product these are the two factors of the same results.
template <typename TYPE, int WN_, int WM_, int NB_, int MB_, bool N_ACROSS, bool M_ACROSS, bool GATED_, int WAVES_EU_>
struct TpShape {
  typedef TYPE Type;
  static constexpr int WN = WN_, WM = WM_, NB = NB_, MB = MB_, THREADS = 64 * WN * WM, BN = 32 * WN * NB, BM = 32 * WM * MB;
  static constexpr bool GATED = GATED_;
  static constexpr int OUT_N = GATED ? BN / 2 : BN, WAVES_EU = WAVES_EU_, GROUPS = (GATED ? NB / 2 : NB) * MB * 4;
  typedef TpStage<BN, N_ACROSS, GATED, THREADS> StageN;
  typedef TpStage<BM, M_ACROSS, false, THREADS> StageM;
  static constexpr int STAGE = StageN::BYTES + StageM::BYTES;
  static_assert(NB % 2 == 0, "two halves");

  __device__ static __forceinline__ int block_n(int i, int wn) { return (i / (NB / 2)) * (BN / 2) + (wn * (NB / 2) + i % (NB / 2)) * 32; }
};

__device__ __forceinline__ float4 tp_four(const fmd_f32x16& v, int q) { return make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]); }
__device__ __forceinline__ int4 tp_four(const tp_i32x16& v, int q) { return make_int4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]); }

template <typename Four>
__device__ __forceinline__ Four tp_sum(const Four* x, int64_t step, int splits) {
  Four s = x[0];
  for (int i = 1; i < splits; ++i) {
    const Four v = x[i * step];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  return s;
}

// of an epilogue that reads nothing more
struct TpNothing {};

struct TpTile {
  int32_t problem, tn, tm;
};

// Tiles in bands of eight rows of tiles, column by column: those that run at once on an XCD (which takes one contiguous run of
// them) share their operands in its L2.
__device__ __forceinline__ TpTile tp_tile(const TpArgs& a, int tile) {
  TpTile t{0, 0, 0};
#pragma unroll
  for (int i = 1; i < kTpProblems; ++i)
    if (i < a.count && tile >= a.p[i].first) t.problem = i;
  const TpProblem& p = a.p[t.problem];
  const int r = tile - p.first, band = 8 * p.tiles_n, b = r / band, in = r - b * band;
  const int rows = min(8, p.tiles_m - 8 * b);
  t.tn = in / rows;
  t.tm = 8 * b + in - t.tn * rows;
  return t;
}

template <typename S, typename Epi>
__global__ void __launch_bounds__(S::THREADS) __attribute__((amdgpu_waves_per_eu(S::WAVES_EU)))
tile_product_kernel(TpArgs a, Epi epi) {
  typedef typename S::Type T;
  typedef typename T::Acc Acc;
  constexpr int NB = S::NB, MB = S::MB;
  __shared__ __attribute__((aligned(1024))) char lds[kTpPlaces * S::STAGE];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wn = wave / S::WM, wm = wave % S::WM;
  int tile, split = 0, splits = 1;
  if ((int)blockIdx.x < a.full) {
    tile = (int)fmd_xcd_block(blockIdx.x, a.full);
  } else {
    const int r = (int)fmd_xcd_block(blockIdx.x - a.full, (int64_t)(a.tiles - a.full) * a.splits);
    splits = a.splits;
    tile = a.full + r / splits;
    split = r % splits;
  }
  const TpTile tt = tp_tile(a, tile);
  const TpProblem& p = a.p[tt.problem];
  const int64_t n0 = (int64_t)tt.tn * S::OUT_N, m0 = (int64_t)tt.tm * S::BM;

  // slices of K of all passes (parts, planes), and those of this workgroup
  const int64_t k_bytes = p.k * T::SIZE;
  const int nk = (int)((k_bytes + kTpSlice - 1) / kTpSlice), passes = p.parts * p.pairs.count;
  const int total = nk * passes;  // at least one: K is not empty
  const int begin = (int)((int64_t)total * split / splits), end = (int)((int64_t)total * (split + 1) / splits);

  typename S::StageN sn;
  typename S::StageM sm;
  sn.place(p.n, n0, p.rows_n, wave, lane);
  sm.place(p.m, m0, p.rows_m, wave, lane);
  int pass = begin / nk, ks = begin - pass * nk;  // of the next slice to copy
  auto open = [&]() {
    const int pair = pass / p.parts, part = pass - pair * p.parts;
    sn.begin(p.n, part, (p.pairs.n >> (2 * pair)) & 3, n0, ks);
    sm.begin(p.m, part, (p.pairs.m >> (2 * pair)) & 3, m0, ks);
  };
  int next = begin;  // slice to copy; past the end zeros, so that every wait counts the same copies
  constexpr int COPIES = S::StageN::LOADS + S::StageM::LOADS;
  auto left = [&]() {
    const int64_t l = k_bytes - (int64_t)ks * kTpSlice;
    return next < end ? (int)(l < kTpSlice ? l : kTpSlice) : 0;
  };
  auto copy_one = [&](const char* place, int j, int left) {
    const uint32_t st = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)place;
    if (j < S::StageN::LOADS)
      sn.copy(st, j, left, wave);
    else
      sm.copy(st + S::StageN::BYTES, j - S::StageN::LOADS, left, wave);
  };
  auto copied = [&]() {
    sn.advance();
    sm.advance();
    ++next;
    if (++ks == nk) {
      ks = 0;
      ++pass;
      if (next < end) open();
    }
  };
  const int ln = S::StageN::lane_at(lane), lm = S::StageM::lane_at(lane);
  tp_i32x4 fn[2][NB], fm[2][MB];
  // the reads of a step, in the order in which the products take them
  constexpr int READS = NB + MB;
  auto read_one = [&](const char* st, int kk, int to, int i) {
    if (i >= 1 && i <= MB)
      fm[to][i - 1] = S::StageM::read(st + S::StageN::BYTES, lm, (wm * MB + i - 1) * 32, kk);
    else
      fn[to][i ? i - MB : 0] = S::StageN::read(st, ln, S::block_n(i ? i - MB : 0, wn), kk);
  };
  Acc acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;

  // A step's products with the next step's reads, and copies, between them, held in this order.
  constexpr int SLOTS = NB * MB;
  auto step = [&](int kk, const char* st, int next_kk, bool copies, const char* place) {
    const int from = kk & 1, to = from ^ 1, rest = copies ? left() : 0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const int slot = i * MB + j;
        acc[i][j] = T::mma(fn[from][i], fm[from][j], acc[i][j]);
#pragma unroll
        for (int r = 0; r < READS; ++r)
          if (r * SLOTS / READS == slot) read_one(st, next_kk, to, r);
        if (copies)
#pragma unroll
          for (int c = 0; c < COPIES; ++c)
            if (c * SLOTS / COPIES == slot) copy_one(place, c, rest);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  // A slice is kTpSteps steps. The operands of a step are read while the one before runs; before the last step every wave has
  // read the whole slice, so its place takes the slice that is kTpPlaces further.
  static_assert((kTpPlaces - 1) * COPIES < 16, "in the low bits of the count");
  auto slice = [&](char* st, char* following) {
#pragma unroll
    for (int kk = 0; kk + 1 < kTpSteps; ++kk) step(kk, st, kk + 1, false, nullptr);
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_waitcnt(tp_wait((kTpPlaces - 2) * COPIES, 0));  // of the slices on their way the first has landed
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    step(kTpSteps - 1, following, 0, true, st);
    copied();
  };
  open();
#pragma unroll
  for (int i = 0; i < kTpPlaces; ++i) {
    const int rest = left();
#pragma unroll
    for (int j = 0; j < COPIES; ++j) copy_one(lds + i * S::STAGE, j, rest);
    copied();
  }
  __builtin_amdgcn_s_waitcnt(tp_wait((kTpPlaces - 1) * COPIES, 15));
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
#pragma unroll
  for (int r = 0; r < READS; ++r) read_one(lds, 0, 0, r);
  for (int s = begin; s < end; s += kTpPlaces)
#pragma unroll
    for (int i = 0; i < kTpPlaces; ++i)
      if (s + i < end) slice(lds + i * S::STAGE, lds + (i + 1) % kTpPlaces * S::STAGE);
  __builtin_amdgcn_s_waitcnt(tp_wait(0, 0));  // no copy outlives the loop

  // a lane's results: row m0 + wm 32 MB + 32 j + lane % 32, four columns from n0 + block + 8 q + 4 (lane / 32)
  if (splits > 1) {
    typedef decltype(tp_four(acc[0][0], 0)) Part;
    Part* out = static_cast<Part*>(a.partial) + (int64_t)((tile - a.full) * splits + split) * (NB * MB * 4) * S::THREADS + t;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          out[((i * MB + j) * 4 + q) * S::THREADS] = tp_four(acc[i][j], q);
        }
    return;
  }
  // Each wave turns its 32 rows at a time round in LDS, so that the epilogue has whole rows side by side in its lanes, and its code
  // once. Chunks of four are permuted by the row: neither the writes (a column of sixteen rows) nor the reads meet a bank twice.
  typedef decltype(tp_four(acc[0][0], 0)) Four;
  constexpr int CHUNKS = NB * 8, REGION = 32 * CHUNKS * 16, EACH = S::GATED ? CHUNKS / 2 : CHUNKS;
  static_assert(REGION * S::THREADS / 64 <= kTpPlaces * S::STAGE, "a place for each wave");
  __syncthreads();
  char* mine = lds + wave * REGION;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int r = lane & 31;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<Four*>(mine + (r * CHUNKS + ((i * 8 + 2 * q + (lane >> 5)) ^ (r & (CHUNKS - 1)))) * 16) = tp_four(acc[i][j], q);
    // What the epilogue reads of memory is asked for some rows ahead of its results: four, or two where four would not fit the registers
    // beside a large tile's sums (they spilt).
    constexpr int AHEAD = S::BN >= 256 && sizeof(typename Epi::Fetch) > 16 ? 2 : 4;
    static_assert(32 * EACH % (64 * AHEAD) == 0, "whole groups");
    for (int k0 = lane; k0 < 32 * EACH; k0 += 64 * AHEAD) {
      int64_t m[AHEAD], n[AHEAD];
      typename Epi::Fetch fetched[AHEAD];
#pragma unroll
      for (int g = 0; g < AHEAD; ++g) {
        const int k = k0 + 64 * g, row = k / EACH, c = k % EACH, half = c / (CHUNKS / 2);
        m[g] = m0 + (wm * MB + j) * 32 + row;
        n[g] = n0 + half * (S::BN / 2) + wn * (NB * 16) + (c - half * (CHUNKS / 2)) * 4;
        fetched[g] = epi.fetch(m[g], n[g]);
      }
#pragma unroll
      for (int g = 0; g < AHEAD; ++g) {
        const int k = k0 + 64 * g, row = k / EACH, c = k % EACH;
        const Four* x = reinterpret_cast<const Four*>(mine) + row * CHUNKS;
        const Four v = x[c ^ (row & (CHUNKS - 1))], u = S::GATED ? x[(c + CHUNKS / 2) ^ (row & (CHUNKS - 1))] : v;
        epi(tt.problem, m[g], n[g], v, u, fetched[g]);
      }
    }
  }
}

// The tiles that several workgroups share: their sums added in order, then the same epilogue. One workgroup per group of four
// results of each thread.
template <typename S, typename Epi>
__global__ void __launch_bounds__(S::THREADS) tile_join_kernel(TpArgs a, Epi epi) {
  constexpr int NB = S::NB, MB = S::MB;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wn = wave / S::WM, wm = wave % S::WM;
  const int rel = blockIdx.x / S::GROUPS, group = blockIdx.x % S::GROUPS;
  const int i = group / (4 * MB), j = group / 4 % MB, q = group % 4;
  const TpTile tt = tp_tile(a, a.full + rel);
  auto sum = [&](int block) {
    typedef decltype(tp_four(typename S::Type::Acc{}, 0)) Four;
    constexpr int64_t step = (int64_t)(NB * MB * 4) * S::THREADS;
    return tp_sum(static_cast<const Four*>(a.partial) + rel * a.splits * step + ((block * MB + j) * 4 + q) * S::THREADS + t, step,
                  a.splits);
  };
  const int64_t m = (int64_t)tt.tm * S::BM + (wm * MB + j) * 32 + (lane & 31);
  const int64_t n = (int64_t)tt.tn * S::OUT_N + S::block_n(i, wn) + 8 * q + 4 * (lane >> 5);
  const auto fetched = epi.fetch(m, n);
  const auto v = sum(i);
  if (S::GATED)
    epi(tt.problem, m, n, v, sum(i + NB / 2), fetched);
  else
    epi(tt.problem, m, n, v, v, fetched);
}

// Host side: sizes, the split of the tiles that do not fill the card, launches.

constexpr int kTpCus = 256;
constexpr int64_t kTpMostTiles = 1 << 22;  // of 512 threads at most: a launch takes fewer than 2^32

// The operand rows of [base, ld elements of `size` bytes]
inline TpOperand tp_operand(const void* a, const void* b, int64_t ld, int64_t plane, int size) {
  return {{static_cast<const char*>(a), static_cast<const char*>(b)}, ld * size, plane * size};
}

struct TpPlan {
  int32_t tiles, full, splits;
  int64_t partial;  // bytes
  float time;       // estimate, us
};

// A shape's measured times (us): of a slice, alone on a CU and by each workgroup of a full one, and of a tile's begin and end. (Fitted to
// products of 16 to 16 875 rows: with tiles chosen by their count alone the float32 block of 16 875 rows of 256 x 680, all gradients, took
// 750 us, by these 571.)
template <typename S>
struct TpTimes {
  static constexpr bool LARGE = S::BN * S::BM >= 65536, SMALL = S::BN * S::BM <= 4096;
  static constexpr float alone = LARGE ? 1.95f : SMALL ? 0.6f : 0.9f, each = LARGE ? 1.95f : SMALL ? 0.31f : 0.69f;
  static constexpr float ends = LARGE ? 12.f : SMALL ? 4.f : 6.f;
};

// Whole rounds of the card run tile by tile; the tiles of the last, partial one may be shared out over the K axis. Of the ways to
// share them the one with the least time by the shape's measured times; `heavy`: of the epilogue, where it reads and writes more
// than the result. (Joining costs a launch and the traffic of the sums.)
template <typename S>
inline TpPlan tp_plan(int64_t tiles, int64_t slices, float heavy) {
  constexpr int64_t per_cu = 4 * S::WAVES_EU * 64 / S::THREADS, round = kTpCus * per_cu, sums = (int64_t)S::NB * S::MB * 16 * S::THREADS * 4;
  typedef TpTimes<S> Times;
  const auto of = [&](int64_t workgroups, float slices) {
    const float k = (float)fmd_cdiv(workgroups, kTpCus);
    const float slice = k * Times::each > Times::alone ? k * Times::each : Times::alone;
    return slices * slice + Times::ends * heavy;
  };
  const int64_t left = tiles % round;
  const float before = (float)(tiles / round) * of(round, (float)slices);
  TpPlan best{(int32_t)tiles, (int32_t)tiles, 1, 0, before + (left ? of(left, (float)slices) : 0.f)};
  for (int64_t s = 2; left && s <= 64 && s <= slices && left * s <= round; ++s) {
    const float traffic = (float)(left * s * sums) * 2.f / 3e6f;
    const float time = before + of(left * s, (float)fmd_cdiv(slices, s)) + 8.f + traffic;
    if (time < 0.95f * best.time) best = {(int32_t)tiles, (int32_t)(tiles - left), (int32_t)s, left * s * sums, time};
  }
  return best;
}

template <typename S, typename Epi>
inline int tp_launch(TpArgs& a, const TpPlan& plan, void* partial, const Epi& epi, hipStream_t stream) {
  a.tiles = plan.tiles;
  a.full = plan.full;
  a.splits = plan.splits;
  a.partial = partial;
  const int shared = plan.tiles - plan.full;
  tile_product_kernel<S, Epi><<<plan.full + shared * plan.splits, S::THREADS, 0, stream>>>(a, epi);
  FMD_CHECK_LAUNCH();
  if (shared) {
    tile_join_kernel<S, Epi><<<shared * S::GROUPS, S::THREADS, 0, stream>>>(a, epi);
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

// the tiles of a problem, numbered after those before it
template <typename S>
inline int64_t tp_tiles(TpProblem& p, int64_t first) {
  p.tiles_n = (int32_t)fmd_cdiv(p.rows_n, S::OUT_N);
  p.tiles_m = (int32_t)fmd_cdiv(p.rows_m, S::BM);
  p.first = (int32_t)first;
  return first + (int64_t)p.tiles_n * p.tiles_m;
}
