// Building blocks of the segment attention kernels: the segment of a tile, tiles of rows staged in LDS, and the
// operands of the matrix instructions.
//
// The query rows of a segment are taken per key head as nq * group packed rows (row r: query r / group, head
// kv * group + r % group), so the query heads that share a key head share its tiles, and the sum over them in the
// gradients of keys and values is part of the product's own sum.
//
// float32 operands are held as three bf16 planes (x3.h: a product is six bf16 products and keeps fp32 accuracy),
// bf16 operands as one.
#pragma once

#include "attention_find.h"
#include "common.h"
#include "x3.h"

typedef short fmd_s16x4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const void *q, *k, *v;                    // rows [tokens, heads, dim], unit stride in dim
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const int64_t *q_off, *k_off;             // [segments + 1]
  int64_t tq, tk;
  int32_t segments, heads, kv_heads, group, dim, causal;
  float scale;
  uint32_t group_mul, group_shift;          // row / group = row * group_mul >> group_shift for rows below 2^31
  uint32_t block0;                          // first workgroup of this launch (launch_ranges)
};

// A launch takes fewer than 2^32 threads a dimension. More workgroups go in several launches, each told its first one:
// launch(workgroups, first).
constexpr int64_t kMostBlocks = 1 << 22;

template <typename Launch>
int launch_ranges(int64_t blocks, const Launch& launch) {
  for (int64_t first = 0; first < blocks; first += kMostBlocks) {
    launch((unsigned)(blocks - first < kMostBlocks ? blocks - first : kMostBlocks), first);
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

__device__ __forceinline__ int attn_token(const AttnArgs& a, int row) {
  return (int)((uint64_t)(uint32_t)row * a.group_mul >> a.group_shift);
}

// What the VJP needs of the forward besides its output. A row's probabilities are exp2(s scale log2(e) - base) inverse; its
// output before rounding is out + residual (bf16: delta = g . o cancels against g . v where few keys count, and the rounding
// of the output alone took the error of gq and gk from 1.4 to 1.7 times that of rounding them).
struct AttnSaved {
  float *base, *inverse;  // [heads, tq]: near the largest scaled score, in log2 units, 1 / row sum (both 0 for a row that sees nothing)
  void* residual;         // bf16 only: [tq, heads, dim]
};

struct AttnBwd {
  const void* g;  // gradient of the output
  int64_t g_row, g_head;
  const void* out;
  AttnSaved saved;
  const float* rows;  // scratch [2, heads, tq]: the exponents' offset and delta (attn_delta_kernel)
};

// The two arrays whose rows are staged in LDS by plain copies: keys and values, or queries and output gradients. bf16: the
// caller's. fp32: their planes [rows, heads, 3, dim], split once for all workgroups that read them (attn_split_kernel).
struct AttnTiles {
  const __bf16 *x, *y;
  int64_t x_row, x_head, y_row, y_head;
};

constexpr int kWaitVm0 = 0 | (7 << 4) | (15 << 8);  // s_waitcnt vmcnt(0)
constexpr float kLog2e = 1.4426950408889634f;

struct AttnSegment {
  int64_t q0, k0;
  int32_t nq, nk;
};

__device__ __forceinline__ AttnSegment attn_segment(const AttnArgs& a, int i) {
  AttnSegment s;
  s.q0 = attn_start(a.q_off, a.segments, a.tq, i);
  s.k0 = attn_start(a.k_off, a.segments, a.tk, i);
  const int64_t nq = attn_start(a.q_off, a.segments, a.tq, i + 1) - s.q0;
  const int64_t nk = attn_start(a.k_off, a.segments, a.tk, i + 1) - s.k0;
  s.nq = nq > 0 ? (int)nq : 0;
  s.nk = nk > 0 ? (int)nk : 0;
  return s;
}

// whether extended segment i is one of the caller's (the first and last have no counterpart on the other side)
__device__ __forceinline__ bool attn_real(const AttnArgs& a, int i) { return i >= 1 && i <= a.segments; }

// ------------------------------------------------------------------------------------ operands

template <int NP>
struct Planes {
  fmd_bf16x8 p[NP];
};

template <typename T>
struct AttnType;
template <>
struct AttnType<__bf16> {
  static constexpr int planes = 1;
};
template <>
struct AttnType<float> {
  static constexpr int planes = 3;
};

// eight values of a row as they lie in memory
template <typename T>
struct Raw8;
template <>
struct Raw8<__bf16> {
  uint4 v;
};
template <>
struct Raw8<float> {
  float4 a, b;
};

template <typename T>
__device__ __forceinline__ Raw8<T> raw_zero() {
  Raw8<T> r;
  __builtin_memset(&r, 0, sizeof(r));
  return r;
}

__device__ __forceinline__ Raw8<__bf16> raw_load(const __bf16* p) { return {*reinterpret_cast<const uint4*>(p)}; }
__device__ __forceinline__ Raw8<float> raw_load(const float* p) {
  return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
}

__device__ __forceinline__ Planes<1> raw_planes(const Raw8<__bf16>& r) {
  Planes<1> o;
  o.p[0] = __builtin_bit_cast(fmd_bf16x8, r.v);
  return o;
}
__device__ __forceinline__ Planes<3> raw_planes(const Raw8<float>& r) {
  fmd_bf16x4 lo[3], hi[3];
  x3_split(r.a, lo[0], lo[1], lo[2]);
  x3_split(r.b, hi[0], hi[1], hi[2]);
  Planes<3> o;
#pragma unroll
  for (int p = 0; p < 3; ++p) o.p[p] = __builtin_shufflevector(lo[p], hi[p], 0, 1, 2, 3, 4, 5, 6, 7);
  return o;
}

__device__ __forceinline__ void planes_of(const float* x, Planes<1>& o) {
#pragma unroll
  for (int e = 0; e < 8; ++e) o.p[0][e] = (__bf16)x[e];
}
__device__ __forceinline__ void planes_of(const float* x, Planes<3>& o) {
  Raw8<float> r = {make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7])};
  o = raw_planes(r);
}

__device__ __forceinline__ fmd_f32x16 mma(const Planes<1>& a, const Planes<1>& b, fmd_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ fmd_f32x16 mma(const Planes<3>& a, const Planes<3>& b, fmd_f32x16 c) {
  return x3_mfma(a.p, b.p, c);
}

__device__ __forceinline__ fmd_f32x16 zero16() {
  fmd_f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// ------------------------------------------------------------------------------------ tiles in LDS

// A tile of ROWS rows of DP values (NP planes), row-major, its 16-byte chunks permuted within a row so that both
// reads are free of conflicts on the 64 banks: the same chunk of sixteen consecutive rows (a quarter of a 16-byte read,
// operands along a row) and four chunks of four consecutive rows (half of a ds_read_b64_tr_b16, operands along a column).
template <int NP, int ROWS, int DP>
struct AttnTile {
  static constexpr int LD = DP == 96 ? 128 : DP;  // a power of two, for the permutation
  static constexpr int CHUNKS = DP / 8, PLANE = ROWS * LD, SIZE = NP * PLANE;

  __device__ static __forceinline__ int at(int row, int chunk) {
    const int high = (row >> 2) & 3;
    const int f = LD == 128 ? ((row & 3) << 2) | high : LD == 64 ? (((row >> 1) & 1) << 2) | high : high;
    return row * LD + ((chunk ^ f) << 3);
  }

  __device__ static __forceinline__ void put(__bf16* s, int row, int chunk, const Planes<NP>& v) {
#pragma unroll
    for (int p = 0; p < NP; ++p) *reinterpret_cast<fmd_bf16x8*>(s + p * PLANE + at(row, chunk)) = v.p[p];
  }

  // A lane's place in the two operand reads. Tiles start at multiples of LD, so the rest of an address is an exclusive or of
  // bits within a row and a constant.
  __device__ static __forceinline__ int lane_rows() {
    const int lane = threadIdx.x & 63;
    return at(lane & 31, lane >> 5);
  }
  __device__ static __forceinline__ int lane_cols() {
    const int lane = threadIdx.x & 63;
    return at(4 * (lane >> 5) + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (lane & 1) * 4;
  }

  // operand of 32 rows (lane: row base + lane % 32) over 16 columns: eight columns from 16 step + 8 (lane / 32);
  // base a multiple of 32
  __device__ static __forceinline__ Planes<NP> rows(const __bf16* s, int lane_at, int base, int step) {
    Planes<NP> o;
#pragma unroll
    for (int p = 0; p < NP; ++p)
      o.p[p] = *reinterpret_cast<const fmd_bf16x8*>(s + p * PLANE + base * LD + (lane_at ^ (step << 4)));
    return o;
  }

  // operand of 32 columns (lane: column 32 block + lane % 32) over the 16 rows from `base` (a multiple of 16), in the order
  // in which a 32 x 32 product holds its rows: for lane half h rows 4 h .. 4 h + 3, then 8 + 4 h .. 8 + 4 h + 3
  __device__ static __forceinline__ Planes<NP> cols(const __bf16* s, int lane_at, int base, int block) {
    Planes<NP> o;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const __bf16* x = s + p * PLANE + base * LD + (lane_at ^ (block << 5));
      const __bf16* y = s + p * PLANE + (base + 8) * LD + (lane_at ^ (block << 5) ^ 16);
      typedef __attribute__((address_space(3))) fmd_s16x4* lds_ptr;
      const fmd_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)x);
      const fmd_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)y);
      o.p[p] = __builtin_bit_cast(fmd_bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return o;
  }
};

// An infinity or a NaN in a row of a tile must not reach a lane that does not see the row, and a weight of zero would not
// keep it out of a matrix product. Tiles that some lane does not see all of (causal calls) are looked through for such rows;
// where there are any, the products take the finite values alone, and a lane that sees such a row has NaN in the columns of the others
// (in a tile that all see, the product leaves NaN or an infinity there).

// bits of the rows (of 32) of a tile that hold a value that is not finite, for the whole wave (of the first plane: what rounds
// to an infinity counts as one)
template <typename Tile>
__device__ __forceinline__ uint32_t rows_not_finite(const __bf16* s) {
  const int lane = threadIdx.x & 63;
  uint32_t over = 0;
  for (int i = lane >> 5; i < Tile::CHUNKS; i += 2) {
    const uint4 v = *reinterpret_cast<const uint4*>(s + Tile::at(lane & 31, i));
    over |= ((v.x & 0x7f807f80u) + 0x00800080u) | ((v.y & 0x7f807f80u) + 0x00800080u) |
            ((v.z & 0x7f807f80u) + 0x00800080u) | ((v.w & 0x7f807f80u) + 0x00800080u);
  }
  const uint64_t b = __ballot((over & 0x80008000u) != 0);
  return (uint32_t)b | (uint32_t)(b >> 32);
}

// whether a product of the wave holds a value that is not finite: as it does wherever one of its operands' rows does
__device__ __forceinline__ bool not_finite(const fmd_f32x16& x, const fmd_f32x16& y) {
  float t = 0.f;
#pragma unroll
  for (int v = 0; v < 16; ++v) t = fmaf(y[v], 0.f, fmaf(x[v], 0.f, t));
  return __any(t != t);
}

// an operand with zeros in the place of values that are not finite
template <int NP>
__device__ __forceinline__ Planes<NP> finite_part(Planes<NP> x) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    uint4 v = __builtin_bit_cast(uint4, x.p[p]);
    auto clean = [](uint32_t w) {
      if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
      if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
      return w;
    };
    v = make_uint4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
    x.p[p] = __builtin_bit_cast(fmd_bf16x8, v);
  }
  return x;
}

// NaN in the sums of every column in which one of `rows` (bits) of a tile holds a value that is not finite, for lanes that see the
// row: from <= row < to. Sums as a 32 x 32 product holds them, a column block each.
template <typename Tile, int DB>
__device__ __forceinline__ void mark_not_finite(fmd_f32x16 (&o)[DB], const __bf16* s, uint32_t rows, int from, int to) {
  const int half = (threadIdx.x & 63) >> 5;
  for (; rows; rows &= rows - 1) {
    const int row = __builtin_ctz(rows);
    const bool sees = row >= from && row < to;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint2 x = *reinterpret_cast<const uint2*>(s + Tile::at(row, 4 * d + r) + 4 * half);
        const uint32_t e[4] = {x.x << 16, x.x, x.y << 16, x.y};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (sees && (e[k] & 0x7f800000u) == 0x7f800000u) o[d][4 * r + k] = NAN;
      }
  }
}

// Rows of a tile on their way to LDS: THREADS threads load NV chunks each (issued together, written after the
// previous tile has been read). Chunks past the rows or past dim are zero: nothing of another segment is read.
template <typename T, int NP, int ROWS, int DP, int THREADS>
struct AttnLoad {
  using Tile = AttnTile<NP, ROWS, DP>;
  static constexpr int N = ROWS * Tile::CHUNKS, NV = (N + THREADS - 1) / THREADS;
  Raw8<T> r[NV];

  // row(i): address of row i of the tile, or null
  template <typename Row>
  __device__ __forceinline__ void load(int t, int dim, const Row& row) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = t + n * THREADS, chunk = i % Tile::CHUNKS;
      const T* p = (N % THREADS == 0 || i < N) && 8 * chunk < dim ? row(i / Tile::CHUNKS) : nullptr;
      r[n] = p ? raw_load(p + 8 * chunk) : raw_zero<T>();
    }
  }
  __device__ __forceinline__ void store(__bf16* s, int t) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = t + n * THREADS;
      if (N % THREADS == 0 || i < N) Tile::put(s, i / Tile::CHUNKS, i % Tile::CHUNKS, raw_planes(r[n]));
    }
  }
};

__device__ __attribute__((aligned(16))) const uint32_t g_attn_zero_chunk[4] = {0, 0, 0, 0};

// Rows of a tile straight into LDS (no register stage): thread t of THREADS fills the 16-byte slots t, t + THREADS, ...
// of the tile, each with the chunk that the permutation puts there. Per lane one 32-bit offset into the tile's rows; the
// chunks past the rows or past dim come from a zero chunk.
template <int NP, int ROWS, int DP, int THREADS>
struct AttnDma {
  using Tile = AttnTile<NP, ROWS, DP>;
  static constexpr int CH = Tile::LD / 8, ACTIVE = THREADS < ROWS * CH ? THREADS : ROWS * CH;  // threads that copy
  static constexpr int N = ROWS * CH / ACTIVE, STEP = ACTIVE / CH;
  static_assert(ROWS * CH % ACTIVE == 0 && ACTIVE % 64 == 0 && ACTIVE % CH == 0, "whole passes of whole waves");

  // thread t's byte offset in the rows of a tile, for even and odd passes (the permutation of rows eight apart differs)
  __device__ static __forceinline__ void offsets(int t, int64_t ld, uint32_t (&off)[2]) {
    const int row0 = t / CH, pos = t % CH;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int chunk = chunk_at(row0 + i * STEP, pos);  // one past DP is never read: any value will do
      off[i] = 2 * (row0 * (uint32_t)ld + 8 * (chunk < Tile::CHUNKS ? chunk : 0));
    }
  }

  // the planes of a tile (plane stride dim)
  __device__ static __forceinline__ void issue(const __bf16* base, int64_t ld, int n, int dim, int t, const uint32_t (&off)[2],
                                               __bf16* lds) {
#pragma unroll
    for (int p = 0; p < NP; ++p) issue_plane(base + p * dim, ld, n, dim, t, off, lds + p * Tile::PLANE);
  }

  // rows [0, n) of the tile at `base` (row stride `ld`), by thread t with its offsets. STEP is a multiple of four rows, and
  // the permutation repeats after sixteen: passes two apart have the same chunks where STEP is a multiple of eight.
  __device__ static __forceinline__ void issue_plane(const __bf16* base, int64_t ld, int n, int dim, int t,
                                                     const uint32_t (&off)[2], __bf16* lds) {
    const int wave_slot = __builtin_amdgcn_readfirstlane(t & ~63);
    if (wave_slot >= ACTIVE) return;
    if (STEP % 8 == 0 && n >= ROWS && dim == DP) {
      const char* p = reinterpret_cast<const char*>(base);  // uniform; a lane adds its 32-bit offset
#pragma unroll
      for (int i = 0; i < N; ++i) {
        copy16(p + off[i & 1], lds + (wave_slot + i * ACTIVE) * 8);
        p += 2 * STEP * ld;
      }
      return;
    }
    asm volatile("" : "+v"(t));  // nothing of the rare path is kept in registers over the caller's loop
    const int row0 = t / CH, pos = t % CH;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = row0 + i * STEP, chunk = chunk_at(row, pos);
      const __bf16* p = base + row * ld + 8 * chunk;
      p = row < n && 8 * chunk < dim ? p : reinterpret_cast<const __bf16*>(g_attn_zero_chunk);
      asm volatile("" : "+v"(p));  // one load instruction with a per-lane address
      copy16(p, lds + (wave_slot + i * ACTIVE) * 8);
    }
  }

  // the chunk that lies at place `pos` of a row (the permutation is its own inverse)
  __device__ static __forceinline__ int chunk_at(int row, int pos) { return (Tile::at(row, pos) - row * Tile::LD) >> 3; }

  // 64 lanes' words to consecutive ones
  __device__ static __forceinline__ void copy4(const float* p, __bf16* to) {
    typedef const __attribute__((address_space(1))) void* global_ptr;
    typedef __attribute__((address_space(3))) void* lds_ptr;
    __builtin_amdgcn_global_load_lds((global_ptr)(uintptr_t)p, (lds_ptr)to, 4, 0, 0);
  }

  __device__ static __forceinline__ void copy16(const void* p, __bf16* to) {
    typedef const __attribute__((address_space(1))) void* global_ptr;
    typedef __attribute__((address_space(3))) void* lds_ptr;
    __builtin_amdgcn_global_load_lds((global_ptr)(uintptr_t)p, (lds_ptr)to, 16, 0, 0);
  }
};

__device__ const float g_attn_no_row[2] = {INFINITY, 0.f};  // offset and delta of a row past the end: exp(s - inf) = 0

// row index of register v of a 32 x 32 product in lane half h
__device__ __forceinline__ int prod_row(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// max over the two lane halves
__device__ __forceinline__ float max_halves(float x) {
  float y = x;
  swap_halves32(x, y);
  return fmaxf(x, y);
}

// sum over aligned groups of LG <= 16 lanes, on the DPP paths
template <int LG>
__device__ __forceinline__ float lanes_sum(float x) {
  if (LG >= 2) x += dpp_read<kDppQuadXor1>(x);
  if (LG >= 4) x += dpp_read<kDppQuadXor2>(x);
  if (LG >= 8) x += dpp_read<kDppHalfMirror>(x);
  if (LG >= 16) x += dpp_read<kDppRowRor8>(x);
  return x;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <>
__device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
template <>
__device__ __forceinline__ void store4<__bf16>(__bf16* p, float a, float b, float c, float d) {
  fmd_bf16x4 v;
  v[0] = (__bf16)a;
  v[1] = (__bf16)b;
  v[2] = (__bf16)c;
  v[3] = (__bf16)d;
  *reinterpret_cast<fmd_bf16x4*>(p) = v;
}

// sixteen bytes past the caches (the `nt` bit) or through them: outputs larger than the last-level cache's share are not
// read again before they are evicted
template <bool NT>
__device__ __forceinline__ void store16(void* p, uint4 v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 x = {v.x, v.y, v.z, v.w};
  if constexpr (NT) __builtin_nontemporal_store(x, static_cast<u32x4*>(p));
  else *static_cast<u32x4*>(p) = x;
}

// eight values of a row, rounded once
template <bool NT, typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    store16<NT>(p, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])));
    store16<NT>(p + 4, make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])));
  } else {
    fmd_bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (__bf16)x[i];
    store16<NT>(p, __builtin_bit_cast(uint4, v));
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const Raw8<T> r = raw_load(p);
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)e[i];
}

// bytes of output from which a call's stores go past the caches (norm and rotation with 205 MB of output 86 us instead of 104,
// the neighbours' VJP with 184 MB 75 instead of 90; with 69 MB 30.3 instead of 27.6)
constexpr int64_t kStreamBytes = 128 << 20;

// the part of eight (four) outputs that their rounding to bf16 dropped
template <typename T, int N>
__device__ __forceinline__ void saved_residual(const AttnSaved& s, int64_t at, const float (&o)[N]) {
  if constexpr (sizeof(T) == 2) {
    if (s.residual) {
      T* p = static_cast<T*>(s.residual) + at;
#pragma unroll
      for (int e = 0; e < N; e += 4)
        store4<T>(p + e, o[e] - (float)(T)o[e], o[e + 1] - (float)(T)o[e + 1], o[e + 2] - (float)(T)o[e + 2],
                  o[e + 3] - (float)(T)o[e + 3]);
    }
  }
}

// attention_rows.hip
template <typename T>
int attn_rows_fwd(const AttnArgs& a, T* out, const AttnSaved& saved, hipStream_t stream);
template <typename T>
int attn_rows_bwd(const AttnArgs& a, const AttnBwd& b, T* gq, T* gk, T* gv, hipStream_t stream);
