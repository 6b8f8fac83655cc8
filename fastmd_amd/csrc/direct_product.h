// Products out[m, n] = sum_k n_op[n, k] m_op[m, k] without a stop in LDS, for few rows m or small matrices: the operands go from
// memory (or the caches) straight into the registers of the matrix instructions. Few rows: the weights are read once, at
// the memory's rate, and nothing is laid out before; small matrices: they stay in the caches, and one launch does what laying out,
// product and join do.
//
// A wave has 16 columns n and 16 MT rows m. Its workgroup's other waves have the next columns (WK 1), or the same ones and
// another part of K each; their sums are then added in order. float32 is split into its three bf16 planes (x3.h) in registers; an m that an
// earlier product left in planes (float32 three, bf16 two) is read so.
#pragma once

#include <type_traits>

#include "direct_shape.h"
#include "tile_product.h"

typedef float dp_f32x4 __attribute__((ext_vector_type(4)));

// One operand: base of each part (for a gated product of the two matrices), elements from a stored row to the next and, where it
// is kept as planes, from a plane to the next; wide: rows and K in whole 16-byte vectors
struct DpOperand {
  const void* base[2];
  int64_t ld, plane;
  int32_t wide;
};

struct DpArgs {
  DpOperand n, m;
  int64_t rows_n, rows_m, k;  // of one part
  int32_t parts, tiles_n, tiles_m;
};

template <typename T>
struct DpType {  // bf16 and float32: bf16 products
  typedef dp_f32x4 Acc;
  typedef float4 Four;
  static constexpr int PLANES = sizeof(T) == 4 ? 3 : 1, UNIT = 32, EACH = 8;  // K of a product, values of a lane
  static constexpr int KEPT = sizeof(T) == 4 ? 3 : 2;                         // planes of what is kept between two products
};
template <>
struct DpType<int8_t> {
  typedef int Acc __attribute__((ext_vector_type(4)));
  typedef int4 Four;
  static constexpr int PLANES = 1, UNIT = 64, EACH = 16, KEPT = 1;
};

// A lane's values of one row (or, across, of one column) as they lie in memory, and as operands. T: float, __bf16, int8_t.
// SPLIT: what is kept in planes of bf16.
template <typename T, bool ACROSS, bool SPLIT>
struct DpLoad {
  static constexpr int EACH = DpType<T>::EACH;
  typedef typename std::conditional<SPLIT, __bf16, T>::type Stored;
  static constexpr int VECTORS = SPLIT ? DpType<T>::KEPT : sizeof(T) == 4 ? 2 : 1, PLANES = SPLIT ? DpType<T>::KEPT : DpType<T>::PLANES;
  tp_i32x4 v[VECTORS];

  // values k .. k + EACH - 1 of row `row`; past `most` is zero
  __device__ __forceinline__ void load(const DpOperand& o, const void* base, int64_t row, int64_t k, int64_t most) {
#pragma unroll
    for (int p = 0; p < VECTORS; ++p) v[p] = tp_i32x4{0, 0, 0, 0};
    if (k >= most) return;
    const Stored* x = static_cast<const Stored*>(base);
    if (ACROSS) {
      Stored e[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) e[i] = x[(k + i < most ? k + i : most - 1) * o.ld + row];
#pragma unroll
      for (int i = 0; i < EACH; ++i) e[i] = k + i < most ? e[i] : (Stored)0;
      __builtin_memcpy(v, e, sizeof(e));
    } else if (SPLIT) {  // always whole vectors, zero past K
#pragma unroll
      for (int p = 0; p < VECTORS; ++p) v[p] = *reinterpret_cast<const tp_i32x4*>(x + p * o.plane + row * o.ld + k);
    } else if (o.wide) {
#pragma unroll
      for (int p = 0; p < VECTORS; ++p) v[p] = reinterpret_cast<const tp_i32x4*>(x + row * o.ld + k)[p];
    } else {
      Stored e[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) e[i] = x[row * o.ld + (k + i < most ? k + i : most - 1)];
#pragma unroll
      for (int i = 0; i < EACH; ++i) e[i] = k + i < most ? e[i] : (Stored)0;
      __builtin_memcpy(v, e, sizeof(e));
    }
  }

  __device__ __forceinline__ void planes(tp_i32x4 (&p)[PLANES]) const {
    if constexpr (sizeof(T) == 4 && !SPLIT) {
      fmd_bf16x4 lo[3], hi[3];
      x3_split(__builtin_bit_cast(float4, v[0]), lo[0], lo[1], lo[2]);
      x3_split(__builtin_bit_cast(float4, v[1]), hi[0], hi[1], hi[2]);
#pragma unroll
      for (int i = 0; i < 3; ++i) p[i] = __builtin_bit_cast(tp_i32x4, __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
#pragma unroll
      for (int i = 0; i < PLANES; ++i) p[i] = v[i];
    }
  }
};

template <typename T, int NP, int MP>
__device__ __forceinline__ typename DpType<T>::Acc dp_mma(const tp_i32x4 (&a)[NP], const tp_i32x4 (&b)[MP], typename DpType<T>::Acc c) {
  if constexpr (std::is_same<T, int8_t>::value) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a[0], b[0], c, 0, 0, 0);
  } else {
    const auto mma = [](tp_i32x4 x, tp_i32x4 y, dp_f32x4 s) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fmd_bf16x8, x), __builtin_bit_cast(fmd_bf16x8, y), s, 0, 0, 0);
    };
    if constexpr (NP == 1 && MP == 2) c = mma(a[0], b[1], c);
    if constexpr (NP == 3) {
      c = mma(a[0], b[2], c);
      c = mma(a[1], b[1], c);
      c = mma(a[2], b[0], c);
      c = mma(a[0], b[1], c);
      c = mma(a[1], b[0], c);
    }
    return mma(a[0], b[0], c);
  }
}

template <typename T, bool N_ACROSS_, bool GATED_, bool M_SPLIT_, int MT_, int WK_>
struct DpShape {
  typedef T Type;
  static constexpr bool N_ACROSS = N_ACROSS_, GATED = GATED_, M_SPLIT = M_SPLIT_;
  static constexpr int MT = MT_, WK = WK_, WAVES = WK > 1 ? WK : 4, THREADS = 64 * WAVES, COLUMNS = WK > 1 ? 16 : 16 * WAVES, ROWS = 16 * MT;
  // operands in planes take more registers: eight units of bf16 ahead spilt (16 rows of 2 048 x 5 504, both products: 33.1 us, 32.4 with four)
  static constexpr int VALUES = (sizeof(T) == 4 || M_SPLIT ? 4 : 8) / (GATED ? 2 : 1);
  static constexpr int AHEAD = VALUES / MT > 0 ? VALUES / MT : 1;  // units on their way
};

template <typename S, typename Epi>
__global__ void __launch_bounds__(S::THREADS) __attribute__((amdgpu_waves_per_eu(S::WK > 1 ? 4 : 2))) direct_product_kernel(DpArgs a, Epi epi) {
  typedef typename S::Type T;
  typedef DpType<T> D;
  constexpr int MT = S::MT, G = S::GATED ? 2 : 1, U = S::AHEAD;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = S::WK > 1 ? wave : 0;
  // the tiles of rows that share columns run together
  const int tm = blockIdx.x % a.tiles_m, tn = blockIdx.x / a.tiles_m;
  const int64_t n0 = (int64_t)tn * S::COLUMNS + (S::WK > 1 ? 0 : 16 * wave), m0 = (int64_t)tm * S::ROWS;
  const int r = lane & 15, q = lane >> 4;
  const int64_t row_n = n0 + r < a.rows_n ? n0 + r : a.rows_n - 1;
  typename D::Acc acc[G][MT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[g][t] = typename D::Acc{0, 0, 0, 0};

  const int per = (int)((a.k + D::UNIT - 1) / D::UNIT), units = per * a.parts;
  for (int first = wk * U; first < units; first += S::WK * U) {
    DpLoad<T, S::N_ACROSS, false> ln[G][U];
    DpLoad<T, false, S::M_SPLIT> lm[MT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int unit = first + u, part = unit >= per && a.parts > 1 ? 1 : 0;
      const int64_t k = unit < units ? (int64_t)(unit - part * per) * D::UNIT + q * D::EACH : a.k;
#pragma unroll
      for (int g = 0; g < G; ++g) ln[g][u].load(a.n, a.n.base[S::GATED ? g : part], row_n, k, a.k);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t row = m0 + 16 * t + r;
        lm[t][u].load(a.m, a.m.base[part], row < a.rows_m ? row : a.rows_m - 1, k, a.k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      tp_i32x4 pn[G][D::PLANES], pm[S::M_SPLIT ? D::KEPT : D::PLANES];
#pragma unroll
      for (int g = 0; g < G; ++g) ln[g][u].planes(pn[g]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        lm[t][u].planes(pm);
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g][t] = dp_mma<T>(pn[g], pm, acc[g][t]);
      }
    }
  }

  // a lane's results: row m0 + 16 t + lane % 16, four columns from n0 + 4 (lane / 16)
  typedef typename D::Four Four;
  if constexpr (S::WK > 1) {
    __shared__ Four sums[S::WK][G * MT][64];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int t = 0; t < MT; ++t) sums[wave][g * MT + t][lane] = __builtin_bit_cast(Four, acc[g][t]);
    __syncthreads();
    for (int t = wave; t < MT; t += S::WK) {
      const int64_t m = m0 + 16 * t + r, n = n0 + 4 * q;
      const auto fetched = epi.fetch(m, n);
      const auto v = tp_sum(&sums[0][t][lane], G * MT * 64, S::WK);
      epi(0, m, n, v, S::GATED ? tp_sum(&sums[0][(G - 1) * MT + t][lane], G * MT * 64, S::WK) : v, fetched);
    }
  } else {
    typename Epi::Fetch fetched[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) fetched[t] = epi.fetch(m0 + 16 * t + r, n0 + 4 * q);
#pragma unroll
    for (int t = 0; t < MT; ++t)
      epi(0, m0 + 16 * t + r, n0 + 4 * q, __builtin_bit_cast(Four, acc[0][t]), __builtin_bit_cast(Four, acc[G - 1][t]), fetched[t]);
  }
}

template <typename S, typename Epi>
inline int dp_launch(DpArgs a, const Epi& epi, hipStream_t stream) {
  a.tiles_n = (int32_t)fmd_cdiv(a.rows_n, S::COLUMNS);
  a.tiles_m = (int32_t)fmd_cdiv(a.rows_m, S::ROWS);
  const int64_t blocks = (int64_t)a.tiles_n * a.tiles_m;
  FMD_REQUIRE(blocks < (int64_t(1) << 22));
  direct_product_kernel<S, Epi><<<(unsigned)blocks, S::THREADS, 0, stream>>>(a, epi);
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

template <typename T, bool N_ACROSS, bool GATED, bool M_SPLIT, typename Epi>
inline int dp_product(const DpArgs& a, const Epi& epi, hipStream_t stream) {
  const DpForm form = dp_form(a.rows_n, a.rows_m, a.k, a.parts, DpType<T>::UNIT);
  const auto with = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    if constexpr (MT == 1)
      if (form.wk == 16) return dp_launch<DpShape<T, N_ACROSS, GATED, M_SPLIT, MT, 16>>(a, epi, stream);
    if (form.wk == 8) return dp_launch<DpShape<T, N_ACROSS, GATED, M_SPLIT, MT, 8>>(a, epi, stream);
    return dp_launch<DpShape<T, N_ACROSS, GATED, M_SPLIT, MT, 1>>(a, epi, stream);
  };
  if (form.mt == 4) return with(std::integral_constant<int, 4>{});
  if (form.mt == 2) return with(std::integral_constant<int, 2>{});
  return with(std::integral_constant<int, 1>{});
}
